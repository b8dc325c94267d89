"""Rows of the cache back as keys and values, against the planes' own bytes in 64 bits."""
import numpy as np
import pytest

from helpers import Twin, orc, pkg

pytestmark = pytest.mark.gpu


def _hadamard(D):
    h = np.ones((1, 1))
    while h.shape[0] < D:
        h = np.block([[h, h], [h, -h]])
    return h / np.sqrt(D)


def _rows64(layer, n):
    """Rows 0 .. n - 1 in the Walsh-Hadamard domain, from the planes and the stage: (K, V), [n, heads, dims] in 64 bits."""
    D, H, S = layer.head_dim, layer.kv_heads, layer.head_dim // 128
    kc, ks, vc, vs = (x.cpu().numpy() for x in (layer.k_code, layer.k_scale, layer.v_code, layer.v_scale))
    stage = layer.stage.cpu().numpy().reshape(2, 2, H, 128, D).astype(np.float64)
    table = layer.table.cpu().numpy()
    K, V = np.zeros((n, H, D)), np.zeros((n, H, D))
    dims = np.arange(D)
    for t in range(n):
        tile, slot, row = t // 128, t // 128 % 2, t % 64
        if (tile + 1) * 128 > n:
            K[t], V[t] = stage[0, slot, :, t % 128], stage[1, slot, :, t % 128]
            continue
        p = table[t // 64]
        code = lambda c: np.stack((c[p, :, row] & 15, c[p, :, row] >> 4), -1).reshape(H, D).astype(np.float64)  # noqa: E731, B023
        per_dim = lambda a, col: a[p][:, dims // (2 * S), col + dims % (2 * S)].astype(np.float64)  # noqa: E731, B023
        per_token = lambda a, col: np.repeat(a[p, :, row, col:col + S].astype(np.float64), 128, -1)  # noqa: E731, B023
        K[t] = (code(kc) * per_dim(ks, 0) + per_dim(ks, 2 * S)) * per_token(ks, 4 * S)
        V[t] = (code(vc) * per_token(vs, 2 * S) + per_token(vs, 3 * S)) * per_dim(vs, 0)
    return K, V


def _check(got, x, dtype):
    """Rounded once from fp32, which is off by log2(D) + 4 roundings of sums at most the sum of the magnitudes."""
    import torch

    D = x.shape[-1]
    want = x @ _hadamard(D)
    slack = np.abs(x).sum(-1, keepdims=True) / np.sqrt(D) * (np.log2(D) + 4) * 2.0 ** -24
    half = torch.finfo(dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= half * (np.abs(want) + slack) + slack + 2.0 ** -25).all(), err.max()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D,H,QH", [(128, 4, 24), (128, 1, 1), (256, 2, 16), (256, 3, 6)])
@pytest.mark.parametrize("n,iters", [(1, 0), (127, 0), (128, 0), (129, 16), (700, 0), (640, 16)])
def test_all_rows_and_ranges(dtype, D, H, QH, n, iters):
    import torch

    tw = Twin(D=D, H=H, QH=QH, capacity_tokens=n, seed=n, dtype=dtype, iters=iters)
    k, v = (orc.synth_kv(n, n, H, D, i) for i in (1, 2))
    tw.append(k, v)
    K, V = _rows64(tw.gpu, n)
    pos = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    gk, gv = tw.gpu.read_rows(0, n, pos)
    _check(gk, K, gk.dtype)
    _check(gv, V, gv.dtype)
    for begin, tokens in ((0, 1), (n - 1, 1), (n // 2, n - n // 2), (n // 3, n // 2)):
        if tokens:
            a, b = tw.gpu.read_rows(begin, tokens, pos)
            assert torch.equal(a, gk[begin:begin + tokens]) and torch.equal(b, gv[begin:begin + tokens])
    assert tw.gpu.errors() == 0


def test_rows_behind_the_newest_and_bad_pages_stay():
    import torch

    n = 400
    tw = Twin(D=128, H=2, QH=4, capacity_tokens=n, seed=1)
    tw.append(*(orc.synth_kv(1, n, 2, 128, i) for i in (1, 2)))
    layer = tw.gpu
    full = layer.read_rows(0, n, torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    for newest in (-1, 0, 255, 256, 299):
        outs = [torch.full((n, 2, 128), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        layer.read_rows(0, n, torch.tensor([newest], dtype=torch.int32, device="cuda"), *outs)
        for out, x in zip(outs, full):
            assert bool((out[newest + 1:] == 7).all())
            sealed = (newest + 1) // 128 * 128
            assert torch.equal(out[:sealed], x[:sealed])
    assert layer.errors() == 0
    # tile 1 at a page that is none: its rows stay, the others come
    for bad, flag in ((layer.pages, pkg().capi.ERR_PAGE_RANGE), (-1, pkg().capi.ERR_PAGE_RANGE)):
        keep = layer.table[3].clone()
        layer.table[3] = bad
        outs = [torch.full((n, 2, 128), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        layer.read_rows(0, n, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), *outs)
        assert layer.errors() == flag
        layer.error_word.zero_()
        layer.table[3] = keep
        for out, x in zip(outs, full):
            assert bool((out[128:256] == 7).all()) and torch.equal(out[:128], x[:128]) and torch.equal(out[256:], x[256:])
    # a table shorter than the sequence
    layer.c.table_len = 4
    outs = [torch.full((n, 2, 128), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    layer.read_rows(0, n, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), *outs)
    assert layer.errors() == pkg().capi.ERR_TABLE_RANGE
    assert bool((outs[0][256:384] == 7).all()) and torch.equal(outs[0][:256], full[0][:256])


@pytest.mark.parametrize("D", [128, 256])
def test_outputs_at_16_bytes_captured_and_on_another_stream(D):
    import torch

    n = 900
    tw = Twin(D=D, H=2, QH=4, capacity_tokens=n, seed=4, dtype=1)
    tw.append(*(orc.synth_kv(1, n, 2, D, i) for i in (1, 2)))
    layer, pos = tw.gpu, torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    want = layer.read_rows(37, 800, pos)
    bufs = [torch.full((800 * 2 * D + 16,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    outs = [b[8:8 + 800 * 2 * D].view(800, 2, D) for b in bufs]  # 16 bytes further
    assert outs[0].data_ptr() % 32 == 16
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            layer.read_rows(37, 800, pos, *outs)
    for _ in range(2):
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(bool((b[:8] == 7).all()) and bool((b[-8:] == 7).all()) for b in bufs)
    assert layer.errors() == 0

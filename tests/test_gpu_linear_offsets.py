"""Linear attention over prompts whose offsets fall: sequences that share rows have more segments than the workspace has places.  Those that do not fit are left alone,
the others are what they are alone, and the memory around the workspace is neither read nor written."""
import ctypes as C

import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


def _i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _call(layer, q, k, v, offsets, reads, writes):
    """(out, errors) with a workspace of the size asked for, in the middle of numbers that would show."""
    import torch

    lib, tokens, batch = pkg().capi.load(), q.shape[0], len(reads)
    n = (lib.kvb_linear_workspace_bytes(tokens, batch, layer.v_heads, layer.head_dim) + 3) // 4
    beside = 256 * layer.v_heads * layer.head_dim ** 2
    ws = torch.full((n + 2 * beside,), float("nan"), dtype=torch.float32, device="cuda")
    ws[:beside] = 7.0
    ws[n + beside:] = 7.0
    out = torch.full((tokens, layer.v_heads, layer.head_dim), 7.0, dtype=layer.dtype, device="cuda")
    off, r, w = _i32(offsets), _i32(reads), _i32(writes)
    pkg().capi.check(lib.kvb_linear_chunk(layer.ref, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), off.data_ptr(), batch, tokens, r.data_ptr(),
                                          w.data_ptr(), C.c_float(0.1), ws[beside:].data_ptr(), out.data_ptr(), None))
    errors = layer.errors()
    layer.error_word.zero_()
    assert bool((ws[:beside] == 7).all()) and bool((ws[n + beside:] == 7).all())
    return out, errors


def _set_up(D, dtype, tokens, batch, vh=4):
    import torch

    g = torch.Generator(device="cuda").manual_seed(tokens)
    layer = pkg().LinearAttention(2, vh, D, torch.tensor([-0.5, -0.01, -0.001, 0.0][:vh]), 2 * batch, dtype=torch.float16 if dtype == "fp16" else torch.bfloat16)
    q, k, v = (torch.randn((tokens, n, D), generator=g, device="cuda").to(layer.dtype) for n in (2, 2, vh))
    first = torch.randn(layer.state.shape, generator=g, device="cuda")
    layer.state.copy_(first)
    return layer, first, q, k, v


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens,times", [(9000, 2), (9000, 4), (2000, 3)])
def test_the_same_rows_again_and_again(D, dtype, tokens, times):
    """Offsets 0, N, 0, N, ...: the sequences between fall and are refused, the first of the others fits and is as it is alone, the last does not fit."""
    import torch

    capi = pkg().capi
    batch = 2 * times - 1
    layer, first, q, k, v = _set_up(D, dtype, tokens, batch)
    reads, writes = list(range(batch)), list(range(batch, 2 * batch))
    want, errors = _call(layer, q, k, v, [0] + [tokens] * batch, reads, writes)
    assert errors == 0
    state = layer.state[batch].clone()
    layer.state.copy_(first)
    out, errors = _call(layer, q, k, v, [0, tokens] * times, reads, writes)
    assert errors == capi.ERR_POSITIONS
    assert torch.equal(layer.state[batch], state)
    changed = [s for s in range(2 * batch) if not torch.equal(layer.state[s], first[s])]
    assert all(s >= batch and (s - batch) % 2 == 0 for s in changed)  # never one that falls
    assert 2 * batch - 1 not in changed
    if changed == [batch]:
        assert torch.equal(out, want)
    assert bool((out != 7).any(-1).all())


@pytest.mark.parametrize("offsets", [[0, 6000, 3000, 9000], [500, 9000, 400, 700], [0, 9000, 8990, 9000]])
def test_sequences_that_share_some_rows(offsets):
    """Each one that is not left alone has the state of its own rows."""
    import torch

    tokens = 9000
    layer, first, q, k, v = _set_up(64, "bf16", tokens, 3)
    _, errors = _call(layer, q, k, v, offsets, [0, 1, 2], [3, 4, 5])
    assert errors == pkg().capi.ERR_POSITIONS
    got = layer.state.clone()
    assert torch.equal(got[:3], first[:3]) and torch.equal(got[4], first[4])
    for s in (0, 2):
        rows = slice(offsets[s], offsets[s + 1])
        layer.state.copy_(first)
        layer.chunk(q[rows], k[rows], v[rows], _i32([0, offsets[s + 1] - offsets[s]]), 0.1, _i32([s]), _i32([s + 3]))
        alone = layer.state[s + 3]
        # other segments, other sums: each side is off by keys of 16 bits, 2^-16 of the sum of the terms' magnitudes, which is up to 2 / pi sqrt(n) = 60 times the state
        # for n terms of a head that keeps everything, and by less in fp32's roundings: 2 * 60 * 2^-16 < 2^-9.  A state of other rows is off by its own size
        assert torch.equal(got[s + 3], first[s + 3]) or float((got[s + 3] - alone).norm() / alone.norm()) < 2.0 ** -8, s
    assert not torch.equal(got[3], first[3]) or not torch.equal(got[5], first[5])

"""What the append that turns keys seals: codes and axes are the format's for the 16-bit rows beside them in the stage, to the bit, with a rounded division by 15, and
the rows are the turned and rotated keys, as a comparison in 64 bits has them."""
import math

import numpy as np
import pytest

from helpers import orc, pkg

pytestmark = pytest.mark.gpu


def _codes(x):
    """Rows [..., n] of fp16 -> their 4-bit codes, step and zero point, in the format's 32-bit arithmetic.  Every operation rounds: numpy on the host divides where a
    device's division by a constant may be a product with its reciprocal, whose step is off by an ulp for about half of the rows."""
    x = x.astype(np.float32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    step = np.maximum((hi - lo) / np.float32(15), np.float32(1e-10))
    q = (x - lo) / step
    whole = np.floor(q)  # halves go up
    code = np.clip(np.where(q - whole >= np.float32(0.5), whole + 1, whole), 0, 15).astype(np.uint8)
    return code, step[..., 0].astype(np.float16), lo[..., 0].astype(np.float16)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,rotary,interleaved,start,T,scaling", [(128, 128, True, 0, 777, {}), (128, 128, False, 100, 1000, dict(scaling="yarn", factor=4.0, original=32768)),
                                                                  (256, 64, False, 16384, 1024, dict(scaling="linear", factor=4.0)), (256, 256, True, 250, 300, {}), (128, 22, True, 5, 251, {})])
def test_sealed_codes_are_those_of_the_rows_in_the_stage(dtype, D, rotary, interleaved, start, T, scaling):
    import torch

    H, QH, S = 4, 24, D // 128
    t16 = torch.float16 if dtype == "fp16" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(T)
    k, v = (torch.randn((T, H, D), generator=g, device="cuda") for _ in range(2))
    for x in (k, v):
        for ch in (3, 17, 64, 101):
            x[..., ch::128] *= 20
    k, v = k.to(t16), v.to(t16)
    pages = 2 * ((start + T + 127) // 128 + 1)
    layer = pkg().KvarnLayer(D, H, QH, pages + 3, torch.from_numpy(orc.shuffled_table(T, pages, pages + 3)), dtype=t16)
    layer.stage.copy_(torch.randn(layer.stage.shape, generator=g, device="cuda"))  # rows of earlier calls
    pos = torch.arange(start, start + T, dtype=torch.int32, device="cuda")
    rope = pkg().Rope(rotary, base=1e6, interleaved=interleaved, **scaling)
    layer.rope_append(rope, k, v, pos)
    assert layer.errors() == 0

    # the rows, turned and rotated in 64 bits; fp32 is off by the turn's cosines and sines (2^-21 of the pair), rotated, and by log2(D) + 2 roundings of sums
    y, slack = k.double(), torch.zeros_like(k, dtype=torch.float64)
    i, j = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    angle = pos.double()[:, None] * rope.inv_freq[None]
    c, s = (rope.factor * f(angle)[:, None] for f in (torch.cos, torch.sin))
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    slack[..., i] = slack[..., j] = (a.abs() + b.abs()) * abs(rope.factor) * 2.0 ** -21
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    while h.shape[0] < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    h /= D ** 0.5
    stage = layer.stage.view(2, 2, H, 128, D)
    last = (start + T - 1) // 128
    first = max(start, (last - 1) * 128)  # the stage has the last two tiles
    at = torch.arange(first, start + T, device="cuda")
    for which, (x, off) in enumerate(((y, slack), (v.double(), slack * 0))):
        want = (x @ h)[first - start:]
        total = ((x.abs().sum(-1, keepdim=True) * (math.log2(D) + 2) * 2.0 ** -24 + off.sum(-1, keepdim=True)) / D ** 0.5)[first - start:]
        got = stage[which, at // 128 % 2, :, at % 128].double()
        assert bool(((got - want).abs() <= 2.0 ** -11 * (want.abs() + total) + total + 2.0 ** -25).all()), "KV"[which]

    # the tiles there that the call has completed
    rows, table = stage.cpu().numpy(), layer.table.cpu().numpy()
    sealed = [tile for tile in (last - 1, last) if tile * 128 >= start // 128 * 128 and (tile + 1) * 128 <= start + T]
    assert sealed
    for tile in sealed:
        p = table[2 * tile:2 * tile + 2]
        unpack = lambda plane: np.stack(((x := plane[p].cpu().numpy().transpose(1, 0, 2, 3).reshape(H, 128, D // 2)) & 15, x >> 4), -1).reshape(H, 128, D)  # noqa: E731, B023
        code, step, low = _codes(rows[0, tile % 2].swapaxes(1, 2))  # K: a row of the matrix is a dim
        assert np.array_equal(unpack(layer.k_code), code.swapaxes(1, 2)), tile
        axes = layer.k_scale[p].cpu().numpy()
        for page in range(2):
            for got, want in ((axes[page, :, :, :2 * S], step), (axes[page, :, :, 2 * S:4 * S], low)):
                assert np.array_equal(got.reshape(H, D).view(np.uint16), want.view(np.uint16)), tile
            assert (axes[page, :, :, 4 * S:] == 1).all()
        code, step, low = _codes(rows[1, tile % 2].reshape(H, 128, S, 128))  # V: a token's slice
        assert np.array_equal(unpack(layer.v_code), code.reshape(H, 128, D)), tile
        axes = layer.v_scale[p].cpu().numpy().transpose(1, 0, 2, 3).reshape(H, 128, 4 * S)
        assert np.array_equal(axes[..., 2 * S:3 * S].view(np.uint16), step.view(np.uint16)) and np.array_equal(axes[..., 3 * S:].view(np.uint16), low.view(np.uint16))
        assert (axes[..., :2 * S] == 1).all()

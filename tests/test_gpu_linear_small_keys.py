"""fp16 keys of any size in linear attention over prompts: the decayed keys that are added to the state keep 22 bits, or 2^-36, however small they are."""
import math

import pytest

from helpers import pkg
from test_gpu_linear import _close, _i32, _wanted

pytestmark = pytest.mark.gpu


def _keys_off(layer, k, v):
    """What the second numbers of decayed keys may miss beside 2^-22 of each, [v_heads, 1, D] of the state, and of what any earlier state was: 2^-36 at the end of a chunk of 64
    tokens, or of a segment of chunks, and no more than the decayed key itself: for either, no more than at the end of the prompt."""
    import torch

    T, share = k.shape[0], layer.v_heads // layer.qk_heads
    g = layer.log_decay.double()
    state = total = 0.0
    for begin in range(0, T, 64):
        rows = slice(begin, min(begin + 64, T))
        most = k[rows].double().abs().amax((0, 2)).repeat_interleave(share)
        sums = v[rows].double().abs().sum(0)[:, None, :]
        off = lambda most: most.clamp_max(2.0 ** -36)[:, None, None] * sums  # noqa: E731, B023
        state, total = state + off(most * torch.exp(g * (T - rows.stop)) if T > rows.stop else most), total + off(most)
    return state, total


def _check(layer, q, k, v, scale, first, out, state, size):
    """test_gpu_linear's bounds, with the keys' second numbers by their own bound instead of 2^-24 of 1."""
    import torch

    o, oo, s, so = _wanted(layer, q, k, v, scale, first)
    T, share = q.shape[0], layer.v_heads // layer.qk_heads
    kept, total = _keys_off(layer, k, v)
    sums = q.double().abs().sum(-1).repeat_interleave(share, 1)[:, :, None]
    oo = oo - scale * 2.0 ** -24 * sums * v.double().abs().sum(0)[None] + scale * sums * total[None, :, 0]
    so = so - 2.0 ** -24 * v.double().abs().sum(0)[:, None, :] + kept
    _close(out, o, oo, "out")
    _close(state, s, so, "state")
    # In the norm, of independent terms: n keys of `size`, decayed, have 1 / (2 |g|) terms' worth of squares; their second numbers are off by 2^-36 / sqrt(3) in the mean
    # square, undecayed, as long as the decayed key is above 2^-37: for ln(2^37 size) / |g| tokens.  The root of 2 ln(2^37 size) / 3 is below 5 for any size here, and
    # heads that keep everything have as many of either.  The rest (22 bits, fp32's sums) stays below 2^-19
    rel = (state.double() - s).flatten(1).norm(dim=1) / s.flatten(1).norm(dim=1)
    assert float(rel.max()) < 2.0 ** -19 + 5 * 2.0 ** -36 / size, rel


def _layer(vh, D):
    import torch

    return pkg().LinearAttention(vh // 2, vh, D, torch.tensor([0.0, -0.02, -0.5, -0.001]).repeat((vh + 3) // 4)[:vh], 2, dtype=torch.float16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,vh", [(256, 80), (700, 4), (2000, 4), (40, 160)])
@pytest.mark.parametrize("size", [1.0, 0.088, 1e-2, 1e-3, 1e-4, 3e-6, 3000.0])
def test_keys_of_one_size(D, T, vh, size):
    import torch

    g = torch.Generator(device="cuda").manual_seed(T + D)
    layer = _layer(vh, D)
    q, k, v = ((torch.randn((T, n, D), generator=g, device="cuda") * x).half() for n, x in ((vh // 2, 1.0), (vh // 2, size), (vh, 1.0)))
    first = torch.randn((vh, D, D), generator=g, device="cuda") * size
    layer.state[0] = first
    scale = D ** -0.5 / size
    out = layer.chunk(q, k, v, _i32([0, T]), scale, _i32([0]), _i32([1]))
    assert layer.errors() == 0
    _check(layer, q, k, v, scale, first, out, layer.state[1], size)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("vh", [80, 4])
@pytest.mark.parametrize("sizes", [[1e-4, 1.0, 100.0, 1e-3, 0.0, 30000.0, 1e-5, 1e-5], [1000.0, 1e-5, 1e-5, 1e-5, 1e-5, 1e-5, 1e-5, 1.0], [0.0] * 5 + [1e-6] * 3])
def test_keys_whose_size_changes(D, vh, sizes):
    """A size for each 64 tokens, up and down by more than fp16 has bits."""
    import torch

    T = 64 * len(sizes) - 11
    g = torch.Generator(device="cuda").manual_seed(T + D)
    layer = _layer(vh, D)
    by_token = torch.tensor(sizes, device="cuda").repeat_interleave(64)[:T, None, None]
    q, v = ((torch.randn((T, n, D), generator=g, device="cuda")).half() for n in (vh // 2, vh))
    k = (torch.randn((T, vh // 2, D), generator=g, device="cuda").clamp(-2, 2) * by_token).half()
    first = torch.randn((vh, D, D), generator=g, device="cuda") * 1e-3
    layer.state[0] = first
    out = layer.chunk(q, k, v, _i32([0, T]), 1e-3, _i32([0]), _i32([1]))
    assert layer.errors() == 0
    o, oo, s, so = _wanted(layer, q, k, v, 1e-3, first)
    kept, _ = _keys_off(layer, k, v)
    _close(layer.state[1], s, so - 2.0 ** -24 * v.double().abs().sum(0)[:, None, :] + kept, "state")
    fits = o.abs() < 65000
    assert bool(((out.double() - o).abs() <= oo)[fits].all())


@pytest.mark.parametrize("vh", [160, 4])
def test_an_infinite_key_beside_large_and_small_ones(vh):
    """Finite keys of its chunk are held as they are, and stay finite."""
    import torch

    T, D = 500, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    layer = pkg().LinearAttention(vh // 2, vh, D, torch.full((vh,), -0.01), 2, dtype=torch.float16)
    q, k, v = ((torch.randn((T, n, D), generator=g, device="cuda") * x).half() for n, x in ((vh // 2, 1e-3), (vh // 2, 1e-3), (vh, 1e-3)))
    k[300] = 60000.0
    k[301, :, 5] = math.inf
    out = layer.chunk(q, k, v, _i32([0, T]), 1e-3, _i32([0]), _i32([1]))
    assert layer.errors() == 0 and bool(torch.isfinite(out[:301]).all())
    state = layer.state[1]
    others = [d for d in range(D) if d != 5]
    assert bool(torch.isfinite(state[:, others]).all()) and not bool(torch.isfinite(state[:, 5]).any())

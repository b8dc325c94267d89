"""fp16 linear attention over prompts where scores or states leave fp16's range on either side: outputs and states as near to 64 bits as in its middle."""
import math

import pytest

from helpers import pkg
from test_gpu_linear import _close, _i32, _wanted
from test_gpu_linear_small_keys import _keys_off

pytestmark = pytest.mark.gpu

# sizes of q, k, v, the state, and the scale that brings outputs to about 1 .. 1000
CASES = {
    "scores of 1e6": (300.0, 300.0, 1.0, 1.0, 1e-6),
    "scores of 1e9": (1e4, 1e4, 1e-2, 1.0, 1e-8),
    "scores of 1e-8": (1e-4, 1e-4, 1.0, 1e-5, 1e7),
    "a state of 1e6": (1.0, 1.0, 1.0, 1e6, 1e-5),
    "a state of 1e20": (1.0, 1.0, 1.0, 1e20, 1e-19),
    "a state of 1e-6": (1.0, 1e-3, 1e-3, 1e-6, 1e5),
    "a state of 1e-20": (1.0, 0.0, 1.0, 1e-20, 1e20),
    "outputs of large and small parts": (100.0, 100.0, 1e3, 1e-2, 1e-6),
}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,vh", [(300, 80), (900, 4), (77, 160)])
@pytest.mark.parametrize("case", list(CASES))
def test_far_from_one(case, T, vh, D):
    import torch

    qs, ks, vs, ss, scale = CASES[case]
    g = torch.Generator(device="cuda").manual_seed(T + D)
    layer = pkg().LinearAttention(vh // 2, vh, D, torch.tensor([0.0, -0.02, -0.5, -0.001]).repeat((vh + 3) // 4)[:vh], 2, dtype=torch.float16)
    q, k, v = ((torch.randn((T, n, D), generator=g, device="cuda").clamp(-4, 4) * x).half() for n, x in ((vh // 2, qs), (vh // 2, ks), (vh, vs)))
    first = torch.randn((vh, D, D), generator=g, device="cuda") * ss
    _run(layer, q, k, v, first, scale)


def _run(layer, q, k, v, first, scale):
    import torch

    T, share = q.shape[0], layer.v_heads // layer.qk_heads
    layer.state[0] = first
    out = layer.chunk(q, k, v, _i32([0, T]), scale, _i32([0]), _i32([1]))
    assert layer.errors() == 0
    # Keys and states times a power of two, the scale by it: the same outputs and bounds, but for test_gpu_linear's allowance for subnormal numbers, which is small then
    up = 2.0 ** (40 - math.frexp(max(float(first.abs().max()), float(k.abs().max())))[1])
    o, oo, s, so = _wanted(layer, q, k.double() * up, v, scale / up, first.double() * up)
    kept, total = _keys_off(layer, k, v)
    sums = q.double().abs().sum(-1).repeat_interleave(share, 1)[:, :, None]
    assert float(o.abs().max()) < 60000
    _close(out, o, oo + scale * sums * total[None, :, 0], "out")
    _close(layer.state[1], s / up, so / up + kept, "state")
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,vh", [(300, 80), (900, 4)])
def test_one_large_row_beside_small_ones(D, T, vh):
    """A key, a query, a value, a row and a column of the state far above the others."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(T + D)
    layer = pkg().LinearAttention(vh // 2, vh, D, torch.tensor([0.0, -0.02, -0.5, -0.001]).repeat((vh + 3) // 4)[:vh], 2, dtype=torch.float16)
    q, k, v = (torch.randn((T, n, D), generator=g, device="cuda").clamp(-4, 4).half() for n in (vh // 2, vh // 2, vh))
    first = torch.randn((vh, D, D), generator=g, device="cuda")
    k[70] *= 1000
    q[100] *= 1000
    v[33] *= 100
    first[:, 5] *= 1e4
    first[:, :, 9] *= 1e5
    _run(layer, q, k, v, first, 1e-8)

"""Infinite keys in linear attention over prompts: the state holds the infinities of the recurrence, and outputs are infinite where its are, with its signs."""
import math

import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


# one segment of several chunks; several segments; steps one after another
@pytest.mark.parametrize("T,vh", [(210, 160), (700, 4), (8, 4)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [0.0, 0.5, 0.999])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_key(D, dtype, T, vh, at, sign):
    import torch

    g = torch.Generator(device="cuda").manual_seed(T + D)
    layer = pkg().LinearAttention(vh // 2, vh, D, torch.full((vh,), -0.05), 2, dtype=torch.float16 if dtype == "fp16" else torch.bfloat16)
    first = torch.randn(layer.state.shape, generator=g, device="cuda")
    layer.state.copy_(first)
    q, k, v = (torch.randn((T, n, D), generator=g, device="cuda").to(layer.dtype) for n in (vh // 2, vh // 2, vh))
    one = torch.ones((), dtype=layer.dtype, device="cuda")
    q, v = torch.where(q == 0, one, q), torch.where(v == 0, one, v)  # 0 times infinity is another matter
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = i32([0, T]), D ** -0.5, i32([0]), i32([1])
    clean = layer.chunk(q, k, v, *args).clone()
    state = layer.state[1].clone()
    row, head, dim = int(at * T), vh // 2 - 1, 7
    k[row, head, dim] = sign * math.inf
    layer.state.copy_(first)
    out = layer.chunk(q, k, v, *args)
    assert layer.errors() == 0
    heads = slice(2 * head, 2 * head + 2)
    # S[dim] = infinity times v from that row on; o = scale q S
    want = sign * math.inf * v[row, heads].float()
    assert torch.equal(layer.state[1, heads, dim], want)
    assert torch.equal(out[row:, heads].float(), q[row:, head, dim, None, None].float() * want[None])
    # nothing else of the head, nor of others, is touched
    keep = torch.ones_like(state, dtype=torch.bool)
    keep[heads, dim] = False
    assert torch.equal(layer.state[1][keep], state[keep])
    assert torch.equal(out[:row], clean[:row])
    others = [h for h in range(vh) if h // 2 != head]
    assert torch.equal(out[:, others], clean[:, others])

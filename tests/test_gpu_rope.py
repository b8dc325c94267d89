"""Rotary positions on the GPU: rows against the formula in 64 bits, the append that turns keys against that formula and, where turns are exact, against the
plain append bit for bit; decode and prefill over keys turned either way."""
import math

import numpy as np
import pytest

from helpers import orc, pkg

pytestmark = pytest.mark.gpu

DTYPES = ["fp16", "bf16"]


def _dtype(name):
    import torch

    return torch.float16 if name == "fp16" else torch.bfloat16


def _pairs(rotary, interleaved):
    """(first dims, second dims) of the pairs."""
    return (list(range(0, rotary, 2)), list(range(1, rotary, 2))) if interleaved else (list(range(rotary // 2)), list(range(rotary // 2, rotary)))


def _turned64(x, pos, inv_freq, factor, rotary, interleaved):
    """Rows turned in 64 bits, and how far fp32 arithmetic may be off before the last rounding: cosine and sine are within 2^-22 (two units
    in the last place of sincospif, half a unit of the reduced angle times pi, the factor's rounding), two products and a sum add 3 * 2^-24."""
    import torch

    x = x.double()
    y, slack = x.clone(), torch.zeros_like(x)
    i, j = _pairs(rotary, interleaved)
    angle = pos.double()[:, None] * inv_freq.double()[None]
    c, s = factor * torch.cos(angle)[:, None], factor * torch.sin(angle)[:, None]
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    slack[..., i] = slack[..., j] = (a.abs() + b.abs()) * abs(factor) * 2.0 ** -21
    return y, slack


def _check(got, y, slack):
    """Rounded once: half a step of the type relative to the value, half the smallest number of fp16, and what fp32 may be off."""
    import torch

    half = torch.finfo(got.dtype).eps / 2
    tol = half * (y.abs() + slack) + slack + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), f"off by {float((err - tol).max()):.3e} beyond the tolerance, {int((err > tol).sum())} values"


def _rope(rotary, interleaved=False, **kw):
    return pkg().Rope(rotary, interleaved=interleaved, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary,behind,shift", [
    (1, 28, 256, 64, 0, 0), (1, 1, 128, 128, 0, 0), (3, 5, 64, 64, 2, 0), (17, 28, 128, 96, 4, 0), (130, 3, 256, 256, 0, 0), (1000, 28, 128, 32, 1, 0),
    (40, 4, 128, 20, 0, 0), (40, 4, 128, 24, 3, 0), (9, 2, 80, 6, 0, 0), (9, 2, 36, 36, 0, 0), (33, 7, 128, 128, 0, 1), (33, 7, 128, 64, 2, 4), (2, 3, 2, 2, 0, 0), (5, 130, 64, 16, 0, 0)])
def test_rows(dtype, interleaved, tokens, heads, dim, rotary, behind, shift):
    import torch

    g = torch.Generator(device="cuda").manual_seed(tokens + rotary)
    wide = torch.zeros((tokens * (heads + behind) * dim + 8), dtype=_dtype(dtype), device="cuda")
    rows = wide[shift:shift + tokens * (heads + behind) * dim].view(tokens, heads + behind, dim)
    rows.copy_(torch.randn(rows.shape, generator=g, device="cuda") * 3)
    x = rows[:, :heads]
    pos = torch.randint(0, 400000, (tokens,), generator=g, device="cuda").to(torch.int32)
    rope = _rope(rotary, interleaved, base=1e6, scaling="yarn", factor=4.0, original=32768)
    y, slack = _turned64(x, pos, rope.inv_freq, rope.factor, rotary, interleaved)
    out = rope.rows(x, pos)
    _check(out, y, slack)
    assert torch.equal(out[..., rotary:], x[..., rotary:])
    # into rows beside those of x in one buffer, and in place: the same bits, nothing else touched
    both = torch.zeros((tokens, 2 * heads + behind + 1, dim), dtype=x.dtype, device="cuda")
    both[:, :heads] = x
    rope.rows(both[:, :heads], pos, out=both[:, heads + 1:2 * heads + 1])
    assert torch.equal(both[:, heads + 1:2 * heads + 1], out) and torch.equal(both[:, :heads], x)
    assert not both[:, heads].any() and not both[:, 2 * heads + 1:].any()
    before = rows[:, heads:].clone()
    rope.rows(x, pos, out=x)
    assert torch.equal(x, out) and torch.equal(rows[:, heads:], before)


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_of_any_size(interleaved):
    """Positions up to the largest and negative ones.  The turns' 53 bits are shared by their whole part: 2 pi * 2^-52 * turns more."""
    import torch

    pos = torch.tensor([0, 1, -1, 378943, -378943, 2**24 + 1, 2**30 + 12345, 2**31 - 1, -2**31], dtype=torch.int32, device="cuda")
    x = torch.randn((len(pos), 3, 128), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    rope = _rope(128, interleaved)
    y, slack = _turned64(x, pos, rope.inv_freq, 1.0, 128, interleaved)
    # the formula's own angle in 64 bits rounds likewise: 2^-53 of the angle for either
    far = pos.double().abs()[:, None, None] * 2.0 ** -50 * x.double().abs().amax()
    _check(rope.rows(x, pos), y, slack + far)
    assert torch.equal(rope.rows(x, pos)[0], x[0])
    back = rope.rows(rope.rows(x, pos[3:4].expand(len(pos)).contiguous()), pos[4:5].expand(len(pos)).contiguous())
    # there and back: two roundings of a pair that keeps its length, each half a step of the larger component at most
    a = x.double().view(len(pos), 3, 64, 2) if interleaved else torch.stack((x[..., :64], x[..., 64:]), -1).double()
    length = (a ** 2).sum(-1, keepdim=True).sqrt().expand_as(a)
    tol = (length.reshape(x.shape) if interleaved else torch.cat((length[..., 0], length[..., 1]), -1)) * (2 ** 0.5 + 1) * 2.0 ** -11 * 1.001 + 2.0 ** -20
    assert bool(((back.double() - x.double()).abs() <= tol).all())


def test_no_tokens_and_values_that_are_not_finite():
    import torch

    rope = _rope(64)
    assert rope.rows(torch.empty((0, 4, 128), dtype=torch.float16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 128)
    x = torch.randn((6, 4, 128), device="cuda").half()
    pos = torch.arange(6, dtype=torch.int32, device="cuda")
    clean = rope.rows(x, pos)
    x[2, 1, 5], x[3, 2, 100] = math.nan, math.inf
    out = rope.rows(x, pos)
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[2, 1, 5] = touched[2, 1, 37] = touched[3, 2, 100] = True
    assert torch.isnan(out[2, 1, [5, 37]]).all() and torch.isinf(out[3, 2, 100]) and torch.equal(out[~touched], clean[~touched])


def _layer(D, H, QH, tokens, dtype, iters=0, seed=0):
    import torch

    n = 2 * ((tokens + 127) // 128 + 1)
    return pkg().KvarnLayer(D, H, QH, n + 3, torch.from_numpy(orc.shuffled_table(seed, n, n + 3)), dtype=_dtype(dtype), sinkhorn_iters=iters)


def _quarter_turned(x, pos, rotary, interleaved, factor_one=1):
    """Rows turned by `pos` quarter turns: exact."""
    import torch

    y = x.clone()
    i, j = _pairs(rotary, interleaved)
    a, b = x[..., i], x[..., j]
    turn = (pos % 4).long()[:, None, None]
    y[..., i] = torch.where(turn == 0, a, torch.where(turn == 1, -b, torch.where(turn == 2, -a, b)))
    y[..., j] = torch.where(turn == 0, b, torch.where(turn == 1, a, torch.where(turn == 2, -b, -a)))
    return y


def _same(a, b):
    return all(bool((getattr(a, n) == getattr(b, n)).all()) for n in ("k_code", "k_scale", "v_code", "v_scale", "stage"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rotary,interleaved,shift", [(128, 128, False, 0), (128, 128, True, 0), (128, 96, False, 0), (128, 40, False, 0), (128, 64, True, 1), (256, 256, False, 0),
                                                         (256, 64, False, 0), (256, 64, True, 0), (256, 22, True, 0), (256, 128, False, 5)])
@pytest.mark.parametrize("before,T,iters", [(0, 1, 0), (127, 1, 0), (100, 40, 0), (0, 130, 0), (90, 300, 0), (120, 140, 3), (0, 64, 16), (77, 6, 16), (0, 777, 0)])
def test_append_of_quarter_turns_is_the_append(dtype, D, rotary, interleaved, shift, before, T, iters):
    """Angles that are whole quarter turns only move values and change signs, so the cache has to be the plain append's of rows turned by hand, bit for
    bit: codes, axes, stage.  Values are never 0, whose cosine of 6e-17 would show."""
    import torch

    H, QH = 2, 6
    g = torch.Generator(device="cuda").manual_seed(D + T)
    k, v, q = (torch.randn((before + T, n, D), generator=g, device="cuda").to(_dtype(dtype)) for n in (H, H, QH))
    k[..., 3] *= 20
    pos = torch.arange(before + T, dtype=torch.int32, device="cuda")
    rope = _rope(rotary, interleaved)
    rope.inv_freq.fill_(math.pi / 2)
    plain, turned = (_layer(D, H, QH, before + T, dtype, iters) for _ in range(2))
    turned_k = _quarter_turned(k, pos, rotary, interleaved)
    if before:
        for layer in (plain, turned):
            layer.append(turned_k[:before].contiguous(), v[:before].contiguous(), pos[:before])
    plain.append(turned_k[before:].contiguous(), v[before:].contiguous(), pos[before:].contiguous())
    # the new rows as a fused projection leaves them, at any 2-byte boundary
    fused = torch.zeros(T * (QH + 2 * H) * D + 8, dtype=q.dtype, device="cuda")[shift:shift + T * (QH + 2 * H) * D].view(T, QH + 2 * H, D)
    fused[:, :QH], fused[:, QH:QH + H], fused[:, QH + H:] = q[before:], k[before:], v[before:]
    kept = fused.clone()
    got = turned.rope_append(rope, fused[:, QH:QH + H], fused[:, QH + H:], pos[before:].contiguous(), q=fused[:, :QH])
    assert _same(plain, turned) and turned.errors() == 0
    assert torch.equal(got, _quarter_turned(q[before:], pos[before:], rotary, interleaved)) and torch.equal(fused, kept)
    # packed rows, queries in place: the same
    again = _layer(D, H, QH, before + T, dtype, iters)
    if before:
        again.append(turned_k[:before].contiguous(), v[:before].contiguous(), pos[:before])
    mine = q[before:].contiguous()
    assert again.rope_append(rope, k[before:].contiguous(), v[before:].contiguous(), pos[before:].contiguous(), q=mine, q_out=mine) is mine
    assert _same(plain, again) and torch.equal(mine, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rotary,interleaved", [(128, 128, False), (128, 64, True), (256, 64, False), (256, 192, True), (128, 30, False)])
@pytest.mark.parametrize("start,T", [(0, 1), (30011, 5), (130000, 100), (64, 50)])
def test_append_stage_against_64_bits(dtype, D, rotary, interleaved, start, T):
    """The stage's rows of the open tile: turn and Walsh-Hadamard rotation in fp32, rounded to fp16 once.  fp32 is off by the turn's slack, rotated
    (every row of the matrix has entries of 1 / sqrt(D)), and by log2(D) + 2 roundings of sums that are at most the sum of magnitudes."""
    import torch

    H, QH = 2, 4
    g = torch.Generator(device="cuda").manual_seed(start + T)
    k, v, q = (torch.randn((T, n, D), generator=g, device="cuda").to(_dtype(dtype)) for n in (H, H, QH))
    k[..., 17] *= 20
    pos = torch.arange(start, start + T, dtype=torch.int32, device="cuda")
    rope = _rope(rotary, interleaved, base=1e6, scaling="ntk", factor=4.0)
    layer = _layer(D, H, QH, start + T, dtype)
    got_q = layer.rope_append(rope, k, v, pos, q=q)
    assert torch.equal(got_q, rope.rows(q, pos))
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    while h.shape[0] < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    y, slack = _turned64(k, pos, rope.inv_freq, rope.factor, rotary, interleaved)
    want = [y @ h / D ** 0.5, v.double() @ h / D ** 0.5]
    total = [(x.abs().sum(-1, keepdim=True) * (math.log2(D) + 2) * 2.0 ** -24 + s.sum(-1, keepdim=True)) / D ** 0.5 for x, s in ((y, slack), (v.double(), slack * 0))]
    stage = layer.stage.view(2, 2, H, 128, D)
    live = (start + T) % 128
    first = max(start, start + T - live)
    for which in range(2):
        rows = stage[which, first // 128 % 2, :, first % 128:(start + T - 1) % 128 + 1].transpose(0, 1).double()
        w, t = want[which][first - start:], total[which][first - start:]
        assert bool(((rows - w).abs() <= 2.0 ** -11 * (w.abs() + t) + t + 2.0 ** -25).all())
    assert layer.errors() == 0


def test_append_leaves_everything_where_positions_are_refused():
    import torch

    layer = _layer(128, 2, 4, 600, "fp16")
    k, v, q = (torch.randn((300, n, 128), device="cuda").half() for n in (2, 2, 4))
    pos = torch.arange(300, dtype=torch.int32, device="cuda")
    pos[299] = 500
    out = torch.full_like(q, 7)
    layer.rope_append(_rope(128), k, v, pos, q=q, q_out=out)
    assert layer.errors() == pkg().capi.ERR_POSITIONS
    assert bool((out == 7).all()) and not layer.stage.any() and not layer.k_code.any() and not layer.v_scale.any()


@pytest.mark.parametrize("start,T", [(0, 600), (100, 900)])
def test_queries_beside_the_append(start, T):
    """So many tiles that the queries are a launch of their own, which starts beside the append: the same queries and cache, and nothing written where the positions
    are refused; what comes next in the stream finds both done."""
    import torch

    D, H, QH = 256, 8, 40
    g = torch.Generator(device="cuda").manual_seed(T)
    k, v, q = (torch.randn((T, n, D), generator=g, device="cuda").bfloat16() for n in (H, H, QH))
    pos = torch.arange(start, start + T, dtype=torch.int32, device="cuda")
    rope = _rope(64, base=1e6)
    one = _layer(D, H, QH, start + T, "bf16")
    one.rope_append(rope, k, v, pos)
    want = rope.rows(q, pos)
    for _ in range(3):
        two = _layer(D, H, QH, start + T, "bf16")  # a new one: an append that begins inside a tile finds other rows there after one that passed it
        mine = q.clone()
        got = two.rope_append(rope, k, v, pos, q=mine, q_out=mine)
        rows = two.read_rows(start, T, pos[-1:])
        assert torch.equal(got, want) and _same(one, two)
        assert all(torch.equal(a, b) for a, b in zip(rows, one.read_rows(start, T, pos[-1:])))
    assert two.errors() == 0
    for bad in (pos.flip(0).contiguous(), pos - start - 1):
        out = torch.full_like(q, 7)
        two.error_word.zero_()
        two.rope_append(rope, k, v, bad, q=q, q_out=out)
        assert two.errors() == pkg().capi.ERR_POSITIONS
        assert bool((out == 7).all()) and _same(one, two)


def test_steps_and_prompts_over_turned_keys():
    """As an engine uses them: a prompt turned with kvb_rope_rows and prefilled, then decode steps whose append turns the key; against attention in 64 bits over
    the same rows.  Tolerance: K and V in 4 bits.  A step of a row's codes is (hi - lo) / 15, a value is off by half of one at most; for rows of
    +-s * 4.5 that is 0.3 s, uniformly spread 0.173 s in the mean square, i.e. scores (q k scale) of standard deviation 0.173 |q| / sqrt(128) ~ 0.173, values
    off by 0.173 of their own size.  Outputs of a softmax over n keys average both: relative error below exp(3 * 0.173) - 1 + 0.173 = 0.86 of a
    single key's value in the worst case, 0.35 in the mean square over rows.  Keys turned the wrong way give unrelated rows: relative error 1.4."""
    import torch

    D, H, QH, T, steps = 128, 2, 8, 700, 70
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v, q = (torch.randn((T + steps, n, D), generator=g, device="cuda").half() for n in (H, H, QH))
    q *= 2.0
    pos = torch.arange(T + steps, dtype=torch.int32, device="cuda")
    rope = _rope(D, base=1e4, scaling="linear", factor=2.0)
    layer = _layer(D, H, QH, T + steps, "fp16")
    scale = 1 / math.sqrt(D)
    outs = [layer.attn_prefill(rope.rows(q[:T], pos[:T]), rope.rows(k[:T], pos[:T]), v[:T].contiguous(), pos[:T], scale, T)]
    for t in range(T, T + steps):
        at = pos[t:t + 1]
        turned = layer.rope_append(rope, k[t:t + 1], v[t:t + 1], at, q=q[t:t + 1])
        outs.append(layer.attn_decode(turned[0], at, scale, t + 1)[None])
    assert layer.errors() == 0
    got = torch.cat(outs).double()
    qt, kt = (_turned64(x, pos, rope.inv_freq, 1.0, D, False)[0] for x in (q, k))
    kt, vt = (x.repeat_interleave(QH // H, 1) for x in (kt, v.double()))
    s = torch.einsum("ihd,jhd->hij", qt, kt) * scale
    s.masked_fill_(torch.ones(s.shape[1:], dtype=torch.bool, device="cuda").triu(1), -math.inf)
    want = torch.einsum("hij,jhd->ihd", s.softmax(-1), vt)
    rel = float(((got - want) ** 2).sum().sqrt() / (want ** 2).sum().sqrt())
    assert rel < 0.35, rel
    # and the rows read back are the keys and values that went in, to the codes' half step
    rk, rv = layer.read_rows(0, T + steps, pos[-1:])
    for back, x in ((rk, kt[:, ::QH // H]), (rv, v.double())):
        assert float(((back.double() - x) ** 2).mean().sqrt() / (x ** 2).mean().sqrt()) < 0.2


def test_captured_and_on_another_stream():
    import torch

    layer = _layer(128, 4, 24, 600, "bf16")
    rope = _rope(128)
    k, v, q = (torch.randn((20, n, 128), device="cuda").bfloat16() for n in (4, 4, 24))
    pos = torch.arange(20, dtype=torch.int32, device="cuda")
    want = layer.rope_append(rope, k, v, pos, q=q).clone()
    stage = layer.stage.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph, out, turned = torch.cuda.CUDAGraph(), torch.empty_like(q), torch.empty_like(q)
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            layer.rope_append(rope, k, v, pos, q=q, q_out=out)
            rope.rows(q, pos, out=turned)
    torch.cuda.synchronize()
    for _ in range(3):
        layer.stage.zero_()
        out.zero_(), turned.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(turned, want) and torch.equal(layer.stage, stage)

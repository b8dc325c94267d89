"""Linear attention with a decay for each head, against its recurrence in 64 bits."""
import math

import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


def _dtype(name):
    import torch

    return torch.float16 if name == "fp16" else torch.bfloat16


def _layer(qk, vh, D, slots, dtype, log_decay=None):
    import torch

    if log_decay is None:  # from next to nothing kept to next to everything, and the ends
        log_decay = -torch.exp2(torch.linspace(3, -9, vh))
        if vh > 2:
            log_decay[0], log_decay[1] = -math.inf, 0.0
    return pkg().LinearAttention(qk, vh, D, log_decay, slots, dtype=_dtype(dtype))


def _wanted(layer, q, k, v, scale, first):
    """One sequence by the quadratic form in 64 bits: (out, state) and how far the kernels may be off.

    A term at a distance of n tokens has the decay's power n: exp is off by 2^-22 (two units in the last place), so its n-th power by n 2^-22, and the
    running product rounds n times; the chunked form's exponent n * log_decay, rounded, is off by n |log_decay| 2^-24 and meets 0 where it is large.
    The products' 16-bit operands: scores, and for the outputs the states' elements, are rounded to the type (half a step: of a score what is left of
    its sum, of a state's element at most the sum of the magnitudes that it came from); keys are split into two numbers of the type that
    hold 16 bits together (bf16; 22 of fp16).  Sums in fp32: 2^-24 a term of what is summed, D terms of a product and 16 partial sums more."""
    import torch

    T, D = q.shape[0], q.shape[2]
    share = layer.v_heads // layer.qk_heads
    q, k, v = q.double().repeat_interleave(share, 1).transpose(0, 1), k.double().repeat_interleave(share, 1).transpose(0, 1), v.double().transpose(0, 1)
    g = layer.log_decay.double()[:, None, None]
    first = first.double()
    n = torch.arange(T, device="cuda", dtype=torch.float64)

    def power(m):  # exp(g m), with nothing kept at -infinity but what is there at distance 0
        return torch.where(m == 0, torch.ones_like(g * 0 + m), torch.exp(torch.where(torch.isinf(g), torch.full_like(g, -1e300), g) * m))

    def off(m):
        return power(m) * (m * (2.0 ** -22 + 2.0 ** -24) + m * torch.where(torch.isinf(g), torch.zeros_like(g), g.abs()) * 2.0 ** -24)

    gap = n[:, None] - n[None, :]
    seen = (gap >= 0).double()
    gap = gap.clamp_min(0)
    s = q @ k.transpose(1, 2)
    out = ((power(gap) * seen * s) @ v + power(n[:, None] + 1) * (q @ first)) * scale
    state = power(torch.full_like(g, T)) * first + (k * power(T - 1 - n[:, None])).transpose(1, 2) @ v
    u = torch.finfo(layer.dtype).eps / 2
    split = 2.0 ** -16 if layer.dtype == torch.bfloat16 else 2.0 ** -21
    sums = (D + 16) * 2.0 ** -24
    mag = q.abs() @ k.abs().transpose(1, 2)
    out_off = ((seen * (power(gap) * (u * s.abs() + (u + split + 2 * sums) * mag) + off(gap) * mag)) @ v.abs()
               + (power(n[:, None] + 1) * (u + split + sums) + off(n[:, None] + 1)) * (q.abs() @ first.abs())) * scale
    # what stays of a state was summed once a chunk or token: roundings of what it held, decayed
    held = (k.abs() * power(T - 1 - n[:, None])).transpose(1, 2) @ v.abs() + power(torch.full_like(g, T)) * first.abs()
    steps = 1 / (1 - torch.exp(g)).clamp_min(1.0 / max(T, 1))  # tokens that a state remembers
    state_off = (k.abs() * off(T - 1 - n[:, None])).transpose(1, 2) @ v.abs() + off(torch.full_like(g, T)) * first.abs() + held * (split + sums + 2 * steps * 2.0 ** -24)
    out_off = out_off + u * out.abs() + scale * 2 * steps * 2.0 ** -24 * (q.abs() @ first.abs() * power(n[:, None] + 1) + (seen * power(gap) * mag) @ v.abs())
    if layer.dtype == torch.float16:  # subnormal outputs, and subnormal second numbers of a split key
        out_off = out_off + 2.0 ** -25 + scale * 2.0 ** -24 * (q.abs().sum(-1, keepdim=True) * v.abs().sum(1, keepdim=True))
        state_off = state_off + 2.0 ** -24 * v.abs().sum(1, keepdim=True)
    return out.transpose(0, 1), out_off.transpose(0, 1), state, state_off


def _inputs(qk, vh, D, tokens, dtype, seed, wide=0, grow=1.0):
    """Rows as parts of wider ones."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    fused = (torch.randn((tokens, 2 * qk + vh + wide, D), generator=g, device="cuda") * grow).to(_dtype(dtype))
    return fused[:, :qk], fused[:, qk:2 * qk], fused[:, 2 * qk:2 * qk + vh]


def _fill(layer, seed):
    import torch

    layer.state.copy_(torch.randn(layer.state.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 4)
    return layer.state.clone()


def _i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _close(got, want, off, what):
    """Within the worst case, value by value; outputs also in the mean square: roundings of three kinds (the output's; scores' and states' beside each other), each
    uniform over at most half a step and independent: sqrt(2 / 3) of half a step together where the two parts do not cancel, 1.2 allowed."""
    import torch

    err = (got.double() - want).abs()
    if got.dtype != torch.float32 and want.numel() > 4096:
        half = torch.finfo(got.dtype).eps / 2
        assert float(err.square().sum().sqrt()) <= 1.2 * half * float(want.square().sum().sqrt()) + 2.0 ** -25 * want.numel() ** 0.5, what
    assert bool((err <= off).all()), f"{what}: {int((~(err <= off)).sum())} values off, by up to {float((err / off.clamp_min(1e-300)).max()):.2f} of the tolerance"


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("qk,vh,D", [(16, 32, 128), (3, 3, 128), (1, 5, 64), (8, 16, 64)])
@pytest.mark.parametrize("batch,wide", [(1, 0), (2, 1), (33, 0), (64, 3)])
def test_decode(dtype, qk, vh, D, batch, wide):
    import torch

    layer = _layer(qk, vh, D, 2 * batch + 1, dtype)
    before = _fill(layer, batch)
    q, k, v = _inputs(qk, vh, D, batch, dtype, 5, wide)
    order = torch.randperm(2 * batch + 1, generator=torch.Generator().manual_seed(batch)).tolist()
    reads, writes = order[:batch], [order[i] if i % 3 == 0 else order[batch + i] for i in range(batch)]  # some in place, some elsewhere
    out = layer.decode(q, k, v, D ** -0.5, _i32(reads), _i32(writes))
    for b in range(batch):
        o, oo, s, so = _wanted(layer, q[b:b + 1], k[b:b + 1], v[b:b + 1], D ** -0.5, before[reads[b]])
        _close(out[b:b + 1], o, oo, f"out {b}")
        _close(layer.state[writes[b]], s, so, f"state {b}")
    for s in set(range(2 * batch + 1)) - set(writes):
        assert torch.equal(layer.state[s], before[s])
    assert layer.errors() == 0


LENGTHS = [[1], [2], [7], [63], [64], [65], [127], [128], [129], [300], [1000], [1, 64, 0, 33, 128, 200, 5], [0, 0, 3], [513, 1, 77], [40] * 12]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("qk,vh,D", [(2, 4, 128), (3, 3, 64)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x))[:30])
def test_chunk(dtype, qk, vh, D, lengths):
    """Sequences packed behind a first row that belongs to none, with two rows behind the last."""
    import torch

    n, tokens = len(lengths), sum(lengths) + 3
    layer = _layer(qk, vh, D, 2 * n, dtype)
    before = _fill(layer, tokens)
    q, k, v = _inputs(qk, vh, D, tokens, dtype, tokens, wide=tokens % 2)
    offsets = [1 + sum(lengths[:b]) for b in range(n + 1)]
    reads, writes = [(5 * b + 1) % n if n % 5 else b for b in range(n)], list(range(n, 2 * n))
    out = torch.full((tokens, vh, D), 7.0, dtype=_dtype(dtype), device="cuda")
    layer.chunk(q, k, v, _i32(offsets), D ** -0.5, _i32(reads), _i32(writes), out=out)
    assert layer.errors() == 0
    assert bool((out[0] == 7).all()) and bool((out[tokens - 2:] == 7).all()) and torch.equal(layer.state[:n], before[:n])
    for b in range(n):
        rows = slice(offsets[b], offsets[b + 1])
        if not lengths[b]:
            assert torch.equal(layer.state[writes[b]], before[reads[b]])
            continue
        o, oo, s, so = _wanted(layer, q[rows], k[rows], v[rows], D ** -0.5, before[reads[b]])
        _close(out[rows], o, oo, f"out {b}")
        _close(layer.state[writes[b]], s, so, f"state {b}")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[193], [256], [320, 1, 641], [1100]])
def test_chunk_with_many_heads(dtype, D, lengths):
    """So many heads that a sequence is one segment of several chunks."""
    import torch

    n, tokens, vh = len(lengths), sum(lengths), 80
    layer = _layer(40, vh, D, n, dtype)
    before = _fill(layer, tokens)
    q, k, v = _inputs(40, vh, D, tokens, dtype, tokens)
    offsets = [sum(lengths[:b]) for b in range(n + 1)]
    slots = _i32(list(range(n)))
    out = layer.chunk(q, k, v, _i32(offsets), D ** -0.5, slots, slots)
    assert layer.errors() == 0
    for b in range(n):
        rows = slice(offsets[b], offsets[b + 1])
        o, oo, s, so = _wanted(layer, q[rows], k[rows], v[rows], D ** -0.5, before[b])
        _close(out[rows], o, oo, f"out {b}")
        _close(layer.state[b], s, so, f"state {b}")


@pytest.mark.parametrize("shift", [0, 1])
def test_outputs_at_any_boundary(shift):
    import torch

    T = 300
    layer = _layer(80, 80, 64, 2, "bf16")
    q, k, v = _inputs(80, 80, 64, T, "bf16", 7)
    buf = torch.full((T * 80 * 64 + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[shift + 8:shift + 8 + T * 80 * 64].view(T, 80, 64)
    layer.chunk(q, k, v, _i32([0, T]), 0.1, _i32([0]), _i32([1]), out=out)
    assert torch.equal(out, layer.chunk(q, k, v, _i32([0, T]), 0.1, _i32([0]), _i32([1])))
    assert bool((buf[:shift + 8] == 7).all()) and bool((buf[shift + 8 + T * 80 * 64:] == 7).all()) and layer.errors() == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_then_steps_is_one_prompt(dtype, D):
    """A prompt in two calls and single tokens behind it, state in place, against the whole in 64 bits; drafts on a copy of the slot leave it alone."""
    import torch

    T, layer = 400, _layer(2, 4, D, 2, dtype)
    q, k, v = _inputs(2, 4, D, T, dtype, 9)
    slot, outs = _i32([0]), []
    for lo, hi in ((0, 130), (130, 390)):
        outs.append(layer.chunk(q[lo:hi], k[lo:hi], v[lo:hi], _i32([0, hi - lo]), D ** -0.5, slot, slot))
    kept = layer.state[0].clone()
    drafts = layer.chunk(q[390:], k[390:], v[390:], _i32([0, 10]), D ** -0.5, slot, _i32([1]))
    assert torch.equal(layer.state[0], kept)
    for t in range(390, 400):
        outs.append(layer.decode(q[t:t + 1], k[t:t + 1], v[t:t + 1], D ** -0.5, slot, slot))
    o, oo, s, so = _wanted(layer, q, k, v, D ** -0.5, torch.zeros_like(kept))
    # a state handed on in fp32 adds nothing that the tolerance does not count
    _close(torch.cat(outs), o, oo, "out")
    _close(drafts, o[390:], oo[390:], "drafts")
    _close(layer.state[0], s, so, "state")
    _close(layer.state[1], s, so, "state of the drafts")


@pytest.mark.parametrize("chunk", [False, True])
def test_what_a_sequence_is_refused_for(chunk):
    """Slots out of range, a slot that two sequences write or that one writes and another reads, offsets that leave the rows: flagged, the sequence left alone, the
    others computed."""
    import torch

    capi = pkg().capi
    D, per = 64, 70 if chunk else 1

    def call(reads, writes, offsets=None, tokens=None):
        n = len(reads)
        layer = _layer(2, 4, D, 6, "bf16")
        before = _fill(layer, 1)
        tokens = n * per if tokens is None else tokens
        q, k, v = _inputs(2, 4, D, tokens, "bf16", 2)
        out = torch.full((tokens, 4, D), 7.0, dtype=torch.bfloat16, device="cuda")
        if chunk:
            layer.chunk(q, k, v, _i32([per * b for b in range(n + 1)] if offsets is None else offsets), 0.1, _i32(reads), _i32(writes), out=out)
        else:
            layer.decode(q, k, v, 0.1, _i32(reads), _i32(writes), out=out)
        done = [bool((out[per * b:per * b + per] != 7).any()) for b in range(n)]
        changed = [s for s in range(6) if not torch.equal(layer.state[s], before[s])]
        return layer.errors(), done, changed

    assert call([0, 1, 2], [3, 4, 5]) == (0, [True] * 3, [3, 4, 5])
    assert call([0, 0, 0], [3, 4, 5]) == (0, [True] * 3, [3, 4, 5])  # a shared prefix
    assert call([0, 1, 2], [0, 1, 2]) == (0, [True] * 3, [0, 1, 2])
    assert call([0, 6, 2], [3, 4, 5]) == (capi.ERR_SLOT, [True, False, True], [3, 5])
    assert call([0, 1, -1], [3, 4, 5]) == (capi.ERR_SLOT, [True, True, False], [3, 4])
    assert call([0, 1, 2], [3, 6, 5]) == (capi.ERR_SLOT, [True, False, True], [3, 5])
    assert call([0, 1, 2], [3, 4, 3]) == (capi.ERR_SLOT, [False, True, False], [4])
    assert call([0, 1, 2], [3, 4, 0]) == (capi.ERR_SLOT, [False, True, False], [4])
    assert call([1, 1, 2], [1, 4, 5]) == (capi.ERR_SLOT, [False, False, True], [5])
    if chunk:
        assert call([0, 1, 2], [3, 4, 5], offsets=[0, 70, 140, 211]) == (capi.ERR_POSITIONS, [True, True, False], [3, 4])
        assert call([0, 1, 2], [3, 4, 5], offsets=[-1, 70, 140, 210])[0] == capi.ERR_POSITIONS
        errors, done, changed = call([0, 1, 2], [3, 4, 5], offsets=[0, 140, 70, 140])
        assert errors == capi.ERR_POSITIONS and changed == [3, 5]


@pytest.mark.parametrize("tokens", [1, 200])
def test_a_head_that_grows_is_refused(tokens):
    import torch

    layer = _layer(2, 4, 64, 1, "bf16", torch.tensor([-0.1, 0.5, math.nan, -0.2]))
    before = _fill(layer, 1)
    q, k, v = _inputs(2, 4, 64, tokens, "bf16", 2)
    out = torch.full((tokens, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    layer.chunk(q, k, v, _i32([0, tokens]), 0.1, _i32([0]), _i32([0]), out=out)
    assert layer.errors() == pkg().capi.ERR_GEOMETRY
    assert bool((out[:, 1:3] == 7).all()) and torch.equal(layer.state[0, 1:3], before[0, 1:3])
    assert bool((out[:, [0, 3]] != 7).any()) and not torch.equal(layer.state[0, [0, 3]], before[0, [0, 3]])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_are_not_finite_reach_later_rows_only(dtype, D, bad):
    """A row's q reaches that row; a row's k or v reaches it and later rows, of its sequence and head."""
    import torch

    T = 210
    layer = _layer(2, 4, D, 4, dtype, torch.full((4,), -0.05))
    before = _fill(layer, 4)
    q, k, v = (x.clone() for x in _inputs(2, 4, D, 2 * T, dtype, 4))
    run = lambda: layer.chunk(q, k, v, _i32([0, T, 2 * T]), D ** -0.5, _i32([0, 1]), _i32([2, 3]))  # noqa: E731
    clean, state = run().clone(), layer.state.clone()
    q[50, 0, 3], k[100, 1, 7], v[150, 0, 9] = bad, bad, bad
    out = run()
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[50, 0:2] = True
    touched[100:T, 2:4] = True
    touched[150:T, 0, 9] = True
    assert torch.equal(out[~touched], clean[~touched])
    assert not torch.isfinite(out[50, 0:2]).any() and not torch.isfinite(out[100:T, 2:4]).any() and not torch.isfinite(out[150:T, 0, 9]).any()
    reached = torch.zeros_like(state, dtype=torch.bool)
    reached[2, 2:4, 7], reached[2, 0, :, 9] = True, True
    assert torch.equal(layer.state[~reached], state[~reached]) and not torch.isfinite(layer.state[reached]).any()
    assert torch.equal(layer.state[:2], before[:2])


def test_captured_with_one_workspace():
    """Two captured chunk calls and a step, replayed: the bits of the calls themselves."""
    import torch

    layer = _layer(4, 8, 128, 4, "bf16")
    q, k, v = _inputs(4, 8, 128, 900, "bf16", 8)
    r, w, off = _i32([0, 1]), _i32([2, 3]), _i32([0, 700, 900])

    def calls():
        a = layer.chunk(q, k, v, off, 0.1, r, w)
        b = layer.chunk(q[:300], k[:300], v[:300], _i32_off, 0.1, w, r)
        return a, b, layer.decode(q[:2], k[:2], v[:2], 0.1, r, r)

    _i32_off = _i32([0, 290, 300])
    first = _fill(layer, 3)
    want = [x.clone() for x in calls()]
    after = layer.state.clone()
    graph = torch.cuda.CUDAGraph()
    layer.state.copy_(first)
    with torch.cuda.graph(graph):
        got = calls()
    for _ in range(3):
        layer.state.copy_(first)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(layer.state, after)


def test_slots_far_into_the_pool():
    """A pool whose offsets pass 2^31 elements."""
    import torch

    layer = _layer(4, 8, 128, 16600, "bf16")  # 16,600 * 8 * 16,384 = 2.18e9 elements
    at = [0, 16599, 16400]
    for s in at:
        layer.state[s].normal_(generator=torch.Generator(device="cuda").manual_seed(s))
    before = [layer.state[s].clone() for s in at]
    q, k, v = _inputs(4, 8, 128, 203, "bf16", 8)
    out = layer.chunk(q, k, v, _i32([0, 1, 3, 203]), 0.1, _i32(at), _i32(at))
    for b, rows in enumerate((slice(0, 1), slice(1, 3), slice(3, 203))):
        o, oo, s, so = _wanted(layer, q[rows], k[rows], v[rows], 0.1, before[b])
        _close(out[rows], o, oo, f"out {b}")
        _close(layer.state[at[b]], s, so, f"state {b}")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[200, 3, 77], [450]])
def test_rows_at_any_boundary(dtype, D, lengths):
    """Rows that start off the 16-byte boundary, and rows an odd number of elements apart: the bits of packed ones."""
    import torch

    n, tokens, qk, vh = len(lengths), sum(lengths), 40, 80
    q, k, v = (x.contiguous() for x in _inputs(qk, vh, D, tokens, dtype, tokens))
    offsets, slots = _i32([sum(lengths[:b]) for b in range(n + 1)]), _i32(list(range(n)))

    def call(q, k, v):
        layer = _layer(qk, vh, D, n, dtype)
        _fill(layer, 5)
        out = layer.chunk(q, k, v, offsets, D ** -0.5, slots, slots)
        assert layer.errors() == 0
        return out, layer.state

    def moved(x, shift, gap):
        stride = x[0].numel() + gap
        buf = torch.zeros(tokens * stride + shift, dtype=x.dtype, device="cuda")
        y = buf[shift:].as_strided(x.shape, (stride, D, 1))
        y.copy_(x)
        return y

    want = call(q, k, v)
    for shift, gap in ((1, 0), (0, 3), (3, 8), (8, 8)):
        got = call(moved(q, shift, gap), moved(k, shift, gap), moved(v, shift, gap))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (shift, gap)


@pytest.mark.parametrize("longest", [8, 60, 300])
def test_as_many_sequences_as_a_call_takes(longest):
    import random

    import torch

    D, vh, rng = 64, 2, random.Random(longest)
    lengths = [rng.randint(0, longest) for _ in range(256)]
    tokens = sum(lengths)
    layer = _layer(1, vh, D, 256, "bf16")
    before = _fill(layer, 1)
    q, k, v = _inputs(1, vh, D, tokens, "bf16", 3)
    slots = torch.randperm(256, generator=torch.Generator().manual_seed(1)).tolist()
    offsets = [sum(lengths[:b]) for b in range(257)]
    out = layer.chunk(q, k, v, _i32(offsets), 0.2, _i32(slots), _i32(slots))
    assert layer.errors() == 0
    for b in range(0, 256, 1 if longest < 100 else 17):
        rows = slice(offsets[b], offsets[b + 1])
        if not lengths[b]:
            assert torch.equal(layer.state[slots[b]], before[slots[b]])
            continue
        o, oo, s, so = _wanted(layer, q[rows], k[rows], v[rows], 0.2, before[slots[b]])
        _close(out[rows], o, oo, f"out {b}")
        _close(layer.state[slots[b]], s, so, f"state {b}")


def test_two_streams_at_once():
    """Calls of two layers on two streams, each with its own workspace: the bits of one after the other."""
    import torch

    sets = []
    for i in range(2):
        layer = _layer(2, 4, 128, 2, "bf16")
        first = _fill(layer, i)
        q, k, v = _inputs(2, 4, 128, 3000, "bf16", 10 + i)
        sets.append((layer, first, q, k, v))
    off, r, w = _i32([0, 3000]), _i32([0]), _i32([1])
    want = []
    for layer, first, q, k, v in sets:
        out = layer.chunk(q, k, v, off, 0.1, r, w)
        want.append((out.clone(), layer.state.clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for (layer, first, q, k, v), stream in zip(sets, streams):
            layer.state[1].zero_()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(layer.chunk(q, k, v, off, 0.1, r, w))
        torch.cuda.synchronize()
        for (layer, *_), g, (out, state) in zip(sets, got, want):
            assert torch.equal(g, out) and torch.equal(layer.state, state) and layer.errors() == 0


def test_same_inputs_same_bits():
    """No sum depends on which CTA or warp comes first."""
    import torch

    layer = _layer(4, 8, 64, 6, "fp16")
    first = _fill(layer, 2)
    q, k, v = _inputs(4, 8, 64, 2000, "fp16", 6)
    args = (q, k, v, _i32([0, 900, 901, 2000]), 0.1, _i32([0, 1, 2]), _i32([3, 4, 5]))
    out, state = layer.chunk(*args).clone(), layer.state.clone()
    for _ in range(5):
        layer.state.copy_(first)
        assert torch.equal(layer.chunk(*args), out) and torch.equal(layer.state, state)


def test_a_captured_call_keeps_its_workspace():
    """A later call that needs a larger workspace, and allocations after it, do not touch what a graph has captured."""
    import torch

    vh, D, few, many = 2, 128, 700, 9000
    layer = _layer(1, vh, D, 2, "bf16")
    first = _fill(layer, 4)
    q, k, v = _inputs(1, vh, D, many, "bf16", 8)
    r, w = _i32([0]), _i32([1])
    args = (q[:few], k[:few], v[:few], _i32([0, few]), 0.1, r, w)
    want, state = layer.chunk(*args).clone(), layer.state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.chunk(*args)
    size = layer.workspace(few, 1).numel()
    layer.chunk(q, k, v, _i32([0, many]), 0.1, r, w)
    assert layer.workspace(many, 1).numel() > size
    others = [torch.full((size,), 3.0, dtype=torch.float32, device="cuda") for _ in range(8)]
    layer.state.copy_(first)
    graph.replay()
    assert torch.equal(out, want) and torch.equal(layer.state, state) and layer.errors() == 0
    assert all(bool((x == 3.0).all()) for x in others)

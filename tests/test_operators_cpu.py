"""The host sides of rotary positions, rows read back and linear attention: frequencies against their formulas, and what is refused before any launch."""
import ctypes as C
import math

import pytest

from helpers import pkg
from test_capi_cpu import _layer


def _frequencies(rotary, base, scaling, factor=1.0, original=0):
    lib = pkg().capi.load()
    host, attention = (C.c_double * (rotary // 2))(), C.c_float()
    assert lib.kvb_rope_frequencies(rotary, base, scaling, factor, original, host, C.byref(attention)) == 0
    return list(host), attention.value


@pytest.mark.parametrize("rotary", [2, 32, 64, 96, 128, 256])
@pytest.mark.parametrize("base", [1e4, 1e6])
def test_frequencies(rotary, base):
    capi = pkg().capi
    plain = [base ** (-2 * p / rotary) for p in range(rotary // 2)]

    def close(got, want):  # a few roundings of pow
        assert len(got) == len(want) and all(abs(a - b) <= 1e-14 * b for a, b in zip(got, want))

    got, factor = _frequencies(rotary, base, capi.ROPE_PLAIN)
    close(got, plain)
    assert factor == 1.0
    got, factor = _frequencies(rotary, base, capi.ROPE_LINEAR, 8.0)
    close(got, [f / 8 for f in plain])
    assert factor == 1.0
    got, factor = _frequencies(rotary, base, capi.ROPE_NTK, 8.0)
    stretched = base * 8.0 ** (rotary / (rotary - 2)) if rotary > 2 else base
    close(got, [stretched ** (-2 * p / rotary) for p in range(rotary // 2)])
    if rotary > 2:  # the last pair is slowed by the factor, the first not at all
        assert abs(got[-1] * 8 / plain[-1] - 1) < 1e-12 and got[0] == 1.0
    got, factor = _frequencies(rotary, base, capi.ROPE_YARN, 8.0, 32768)
    assert abs(factor - (0.1 * math.log(8) + 1)) < 1e-7
    for p, (f, g) in enumerate(zip(plain, got)):
        turns = 32768 * f / (2 * math.pi)
        assert f / 8 * (1 - 1e-12) <= g <= f * (1 + 1e-12)
        # the ramp's ends lie on whole pairs, so one pair of leeway beside 32 turns and beside one
        ratio = base ** (2 / rotary)
        if turns > 32 * ratio:
            assert abs(g / f - 1) < 1e-12
        if turns < 1 / ratio and p < rotary // 2:
            assert abs(g * 8 / f - 1) < 1e-12


def test_frequencies_refused():
    capi = pkg().capi
    lib = capi.load()
    host, a = (C.c_double * 64)(), C.c_float()

    def call(rotary=128, base=1e4, scaling=0, factor=1.0, original=0, out=host):
        return lib.kvb_rope_frequencies(rotary, base, scaling, factor, original, out, C.byref(a))

    assert call() == capi.KVB_OK
    for bad in (dict(rotary=0), dict(rotary=127), dict(rotary=-2), dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(scaling=4), dict(scaling=-1),
                dict(scaling=1, factor=0.5), dict(scaling=2, factor=math.nan), dict(scaling=3, factor=2.0), dict(out=None)):
        assert call(**bad) == capi.KVB_EINVAL, bad
    with pytest.raises(ValueError):
        pkg().Rope(64, scaling="other", device="cpu")
    with pytest.raises(capi.KvarnError):
        pkg().Rope(63, device="cpu")


def _rope(capi, **over):
    R = capi.kvb_rope(inv_freq=1 << 20, factor=1.0, rotary_dim=64, interleaved=0)
    for k, v in over.items():
        setattr(R, k, v)
    return R


MIB = 1 << 20


def test_rope_rows_refused():
    capi = pkg().capi
    lib = capi.load()
    R = _rope(capi)

    def call(R=R, x=16 * MIB, xs=1024, out=32 * MIB, os=1024, pos=64 * MIB, tokens=4, heads=8, dim=128, dtype=0):
        return lib.kvb_rope_rows(None if R is None else C.byref(R), x, xs, out, os, pos, tokens, heads, dim, dtype, None)

    assert call(tokens=0) == capi.KVB_OK
    for bad in (dict(R=None), dict(R=_rope(capi, inv_freq=None)), dict(R=_rope(capi, inv_freq=(1 << 20) + 4)), dict(R=_rope(capi, rotary_dim=63)), dict(R=_rope(capi, rotary_dim=0)), dict(R=_rope(capi, rotary_dim=130)),
                dict(R=_rope(capi, interleaved=2)), dict(R=_rope(capi, factor=math.nan)), dict(x=None), dict(out=None), dict(pos=None), dict(tokens=-1), dict(heads=0), dict(dim=0),
                dict(dtype=2), dict(xs=1023), dict(os=1000),
                dict(out=16 * MIB + 16),             # beside x, not x itself
                dict(out=16 * MIB, os=2048),         # x itself at another distance
                dict(xs=1100, os=1100, out=16 * MIB + 2 * 100),  # the distance does not hold both
                dict(pos=32 * MIB + 64), dict(R=_rope(capi, inv_freq=32 * MIB + 512))):
        assert call(**bad) == capi.KVB_EINVAL, bad
    assert call(heads=5000, xs=1 << 20, os=1 << 20, out=1 << 34) == capi.KVB_ERANGE


def test_rope_append_refused():
    capi = pkg().capi
    lib = capi.load()
    L = _layer(capi)

    def call(L=L, R=_rope(capi), q=16 * MIB, qs=3200, qo=32 * MIB, qos=3200, k=48 * MIB, ks=512, v=64 * MIB, vs=512, pos=80 * MIB, tokens=4):
        return lib.kvb_rope_append(C.byref(L), C.byref(R), q, qs, qo, qos, k, ks, v, vs, pos, tokens, None)

    assert call(tokens=0) == capi.KVB_OK
    for bad in (dict(L=_layer(capi, kv_heads=9)), dict(L=_layer(capi, stage=None)), dict(R=_rope(capi, rotary_dim=130)), dict(R=_rope(capi, inv_freq=None)), dict(k=None), dict(v=None),
                dict(pos=None), dict(tokens=-1), dict(q=None), dict(qo=None), dict(ks=511), dict(vs=0), dict(qs=2000), dict(qos=1),
                dict(qo=16 * MIB + 32), dict(qo=48 * MIB), dict(qo=64 * MIB - 64), dict(qo=80 * MIB - 64), dict(R=_rope(capi, inv_freq=32 * MIB + 8)),
                # a fused projection's rows: queries, keys and values beside each other, the output over the keys
                dict(q=16 * MIB, qs=4096, k=16 * MIB + 2 * 3200, ks=4096, v=16 * MIB + 2 * 3600, vs=4096, qo=16 * MIB + 64, qos=4096)):
        assert call(**bad) == capi.KVB_EINVAL, bad


def test_read_rows_refused():
    capi = pkg().capi
    lib = capi.load()

    def call(L=_layer(capi), begin=0, tokens=100, pos=16 * MIB, k=32 * MIB, v=48 * MIB):
        return lib.kvb_read_rows(C.byref(L), begin, tokens, pos, k, v, None)

    assert call(tokens=0) == capi.KVB_OK
    for bad in (dict(L=_layer(capi, head_dim=64)), dict(L=_layer(capi, stage=None)), dict(begin=-1), dict(tokens=-5), dict(begin=2**31 - 50), dict(pos=None), dict(k=None), dict(v=None),
                dict(k=32 * MIB + 2), dict(v=48 * MIB + 8), dict(v=32 * MIB + 1024)):
        assert call(**bad) == capi.KVB_EINVAL, bad


def _linear(capi, **over):
    L = capi.kvb_linear(state=1 << 32, log_decay=16, slots=4, qk_heads=4, v_heads=8, head_dim=128, dtype=1, error_word=None)
    for k, v in over.items():
        setattr(L, k, v)
    return L


def test_linear_refused():
    capi = pkg().capi
    lib = capi.load()

    def call(L=_linear(capi), chunk=True, q=16 * MIB, qs=512, k=32 * MIB, ks=512, v=48 * MIB, vs=1024, offsets=16, batch=2, tokens=100, reads=16, writes=16, out=64 * MIB):
        if chunk:
            return lib.kvb_linear_chunk(C.byref(L), q, qs, k, ks, v, vs, offsets, batch, tokens, reads, writes, 0.1, 96 * MIB, out, None)
        return lib.kvb_linear_decode(C.byref(L), q, qs, k, ks, v, vs, batch, reads, writes, 0.1, out, None)

    for chunk in (False, True):
        assert call(batch=0, chunk=chunk) == capi.KVB_OK
        for bad in (dict(L=_linear(capi, state=None)), dict(L=_linear(capi, log_decay=None)), dict(L=_linear(capi, state=(1 << 32) + 4)), dict(L=_linear(capi, head_dim=256)),
                    dict(L=_linear(capi, head_dim=32)), dict(L=_linear(capi, v_heads=6)), dict(L=_linear(capi, qk_heads=0)), dict(L=_linear(capi, v_heads=2)),
                    dict(L=_linear(capi, v_heads=512)), dict(L=_linear(capi, slots=0)), dict(L=_linear(capi, dtype=2)), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
                    dict(reads=None), dict(writes=None), dict(batch=-1), dict(qs=511), dict(ks=0), dict(vs=1023), dict(out=16 * MIB), dict(out=32 * MIB), dict(out=48 * MIB),
                    dict(out=(1 << 32) + 4096)):
            assert call(**bad, chunk=chunk) == capi.KVB_EINVAL, (chunk, bad)
        assert call(batch=257, chunk=chunk) == capi.KVB_ERANGE
    assert call(offsets=None) == capi.KVB_EINVAL
    assert call(tokens=-1) == capi.KVB_EINVAL
    assert lib.kvb_linear_workspace_bytes(8192, 1, 32, 128) > 0


def test_python_refuses_rows_that_are_not_rows():
    import torch

    from importlib import import_module

    pkg()
    row_stride = import_module("kvarn_b200.cache").row_stride
    x = torch.zeros((5, 7, 128), dtype=torch.float16)
    assert row_stride(x, 7, 128, torch.float16, 5) == 7 * 128
    assert row_stride(x[:, :3], 3, 128, torch.float16, 5) == 7 * 128
    for bad in ((x.bfloat16(), 7, 128), (x, 6, 128), (x, 7, 64), (x[0], 7, 128), (x.transpose(0, 1), 5, 128), (x[..., ::2], 7, 64), (x[:, ::2], 4, 128), (x[:4], 7, 128)):
        with pytest.raises(ValueError):
            row_stride(*bad, torch.float16, 5)
    check_indices = import_module("kvarn_b200.cache").check_indices
    at = torch.arange(8, dtype=torch.int32)
    assert check_indices(at, 8, "x") == at.data_ptr() and check_indices(at[3:4], 1, "x") == at[3:].data_ptr() and check_indices(at[:0], 0, "x") is not None
    for bad in ((at, 7), (at.long(), 8), (at[::2], 4), (at.view(2, 4), 8)):
        with pytest.raises(ValueError):
            check_indices(*bad, "x")


def test_tensors_off_the_device_are_refused():
    """Rows, indices and layers in host memory: a ValueError before the library sees an address."""
    import torch

    p = pkg()
    rope = p.Rope(64, device="cpu")
    x, at = torch.zeros(2, 4, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        rope.rows(x, at)
    layer = p.KvarnLayer(128, 4, 8, 4, torch.arange(4, dtype=torch.int32), device="cpu")
    with pytest.raises(ValueError, match="device"):
        layer.rope_append(rope, x, x, at)
    with pytest.raises(ValueError, match="device"):
        layer.rope_append(rope, x, x, at, q=torch.zeros(2, 8, 128, dtype=torch.float16))
    with pytest.raises(ValueError, match="device"):
        layer.read_rows(0, 2, at[:1])
    mix = p.LinearAttention(4, 4, 128, torch.zeros(4), 2, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="device"):
        mix.decode(x, x, x, 1.0, at, at)
    with pytest.raises(ValueError, match="device"):
        mix.chunk(x, x, x, torch.zeros(3, dtype=torch.int32), 1.0, at, at)

"""Linear attention over prompts where a warp's wait gives up at once while tiles and products of others are under way: reported, nothing written but outputs
and states that are right, and the call behind it is as if nothing had been.  The kernels are built for it: no wait of the library is made to run out."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from helpers import ROOT, pkg

pytestmark = pytest.mark.gpu

# by role, each alone and all together: state, row and score warps, the two MMA warps, the load and the store warp
WARPS = {"all": 0xFFFFFF, "state": 0xFF, "one state warp": 1 << 3, "rows": 0xFF00, "one row warp": 1 << 9, "scores": 0x330000, "one score warp": 1 << 20, "state products": 1 << 18,
         "row products": 1 << 22, "loads": 1 << 19, "stores": 1 << 23}


@pytest.fixture(scope="module")
def gives_up(tmp_path_factory):
    if shutil.which("nvcc") is None:
        pytest.skip("needs nvcc on the GPU machine")
    home = os.path.join(ROOT, "ninfer-3080-iq3_s_b200")
    pkg().capi.load()
    lib = str(tmp_path_factory.mktemp("gives_up") / "liblinear.so")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", "-I", os.path.join(home, "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "linear_gives_up.cu"), "-o", lib, "-L", home, "-lkvarn_b200", "-Xlinker", "-Bsymbolic", "-Xlinker", "-rpath", "-Xlinker", home],
                   check=True)
    return C.CDLL(lib)


# one segment of several chunks; one of two, where every load is under way at once; several segments and launches; rows that TMA does not take
@pytest.mark.parametrize("dtype,D,vh,tokens,shift", [("bf16", 128, 80, 1000, 0), ("fp16", 64, 80, 900, 0), ("fp16", 128, 80, 120, 0), ("bf16", 64, 4, 2000, 0), ("bf16", 128, 80, 700, 1)])
@pytest.mark.parametrize("parity", [0, 1])
@pytest.mark.parametrize("who", list(WARPS))
def test_a_call_that_gives_up(gives_up, who, parity, dtype, D, vh, tokens, shift):
    import torch

    g = torch.Generator(device="cuda").manual_seed(tokens)
    layer = pkg().LinearAttention(vh // 2, vh, D, -torch.exp2(torch.linspace(-2, -9, vh)), 2, dtype=torch.float16 if dtype == "fp16" else torch.bfloat16)
    first = torch.randn(layer.state.shape, generator=g, device="cuda")
    q, k, v = (torch.randn((tokens * n * D + 8,), generator=g, device="cuda").to(layer.dtype)[shift:shift + tokens * n * D].view(tokens, n, D) for n in (vh // 2, vh // 2, vh))
    off, r, w = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, tokens], [0], [1]))
    ws = layer.workspace(tokens, 1)
    buf = torch.empty(v.numel() + 16, dtype=v.dtype, device="cuda")

    def call(lib):
        buf.fill_(7.0)
        layer.state.copy_(first)
        layer.error_word.zero_()
        torch.cuda.synchronize()
        assert lib.kvb_linear_chunk(layer.ref, C.c_void_p(q.data_ptr()), C.c_int64(q.stride(0)), C.c_void_p(k.data_ptr()), C.c_int64(k.stride(0)), C.c_void_p(v.data_ptr()),
                                    C.c_int64(v.stride(0)), C.c_void_p(off.data_ptr()), 1, tokens, C.c_void_p(r.data_ptr()), C.c_void_p(w.data_ptr()), C.c_float(0.1),
                                    C.c_void_p(ws.data_ptr()), C.c_void_p(buf[8:].data_ptr()), None) == 0
        torch.cuda.synchronize()
        assert torch.all(buf[:8] == 7.0) and torch.all(buf[-8:] == 7.0) and torch.equal(layer.state[0], first[0])
        return buf[8:-8].clone(), layer.state[1].clone(), layer.errors()

    library = pkg().capi.load()
    out, state, errors = call(library)
    assert errors == 0 and torch.isfinite(out).all() and torch.isfinite(state).all()
    assert gives_up.set_gives_up(C.c_uint32(WARPS[who]), C.c_uint32(parity)) == 0
    got, after, errors = call(gives_up)
    assert errors in (0, pkg().capi.ERR_WAIT_TIMEOUT)
    if errors == 0:  # a short call has no wait for such a phase; loads wait for a stage from the fourth chunk on
        assert (parity == 1 or (who == "loads" and (tokens < 4 * 64 or vh < 80))) and torch.equal(got, out) and torch.equal(after, state)
    elif vh == 80:  # (sums of segments that were given up go into later segments)
        assert bool(((got == out) | (got == 7.0)).all())
        assert bool(((after == state) | (after == first[1])).all())
    assert gives_up.set_gives_up(C.c_uint32(0), C.c_uint32(0)) == 0
    for lib in (gives_up, library):
        got, after, errors = call(lib)
        assert errors == 0 and torch.equal(got, out) and torch.equal(after, state)

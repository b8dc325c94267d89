"""Rows read back where the wait for a CTA's first tile, or for a later one, gives up at once while tiles are on their way: reported, the rows of that tile and of
those behind it are left as they are, and the call behind it is as if nothing had been.  The kernel is built for it: no wait of the library is made to run out."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from helpers import ROOT, Twin, orc, pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def builds(tmp_path_factory):
    if shutil.which("nvcc") is None:
        pytest.skip("needs nvcc on the GPU machine")
    home = os.path.join(ROOT, "ninfer-3080-iq3_s_b200")
    pkg().capi.load()
    made = {}
    for tile in (0, 1, 2):
        lib = str(tmp_path_factory.mktemp("gives_up") / ("libread_%d.so" % tile))
        made[tile] = lib, subprocess.Popen(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
                                            "-DKVB_READ_PROBES=(n<%d?kSpinLimit:0u)" % tile, os.path.join(home, "csrc", "kvb_read.cu"), "-o", lib, "-L", home, "-lkvarn_b200",
                                            "-Xlinker", "-Bsymbolic", "-Xlinker", "-rpath", "-Xlinker", home])
    for lib, build in made.values():
        assert build.wait() == 0
    return {tile: C.CDLL(lib) for tile, (lib, _) in made.items()}


@pytest.mark.parametrize("D,H,T", [(128, 8, 700), (128, 8, 20011), (256, 8, 15000), (128, 1, 100)])
@pytest.mark.parametrize("tile", [0, 1, 2])
def test_a_read_that_gives_up(builds, tile, D, H, T):
    import torch

    tw = Twin(D=D, H=H, QH=H, capacity_tokens=T, seed=T)
    at = torch.arange(T, dtype=torch.int32, device=tw.dev)
    tw.gpu.append(*(torch.from_numpy(orc.synth_kv(T, T, H, D, i)).to(tw.dev) for i in (1, 2)), at)
    rows = T * H * D
    bufs = [torch.empty(rows + 32, dtype=torch.float16, device=tw.dev) for _ in range(2)]

    def call(lib):
        for b in bufs:
            b.fill_(7.0)
        assert lib.kvb_read_rows(C.byref(tw.gpu.c), 0, T, C.c_void_p(at[T - 1:].data_ptr()), C.c_void_p(bufs[0][16:].data_ptr()), C.c_void_p(bufs[1][16:].data_ptr()), None) == 0
        torch.cuda.synchronize()
        assert all(torch.all(b[:16] == 7.0) and torch.all(b[-16:] == 7.0) for b in bufs)
        errors = tw.gpu.errors()
        tw.gpu.error_word.zero_()
        return [b[16:-16].view(T, H, D).clone() for b in bufs], errors

    library = pkg().capi.load()
    want, errors = call(library)
    assert errors == 0
    got, errors = call(builds[tile])
    # as many CTAs a head of K or V as are resident at once: the tiles of the first `tile` rounds are there
    step = torch.cuda.get_device_properties(0).multi_processor_count * (3 if D == 256 else 4) // (2 * H)
    done = min(T, tile * step * 128)
    assert errors == (0 if done == T else pkg().capi.ERR_WAIT_TIMEOUT)
    for a, b in zip(got, want):
        assert torch.equal(a[:done], b[:done]) and torch.all(a[done:] == 7.0)
    got, errors = call(library)
    assert errors == 0 and all(torch.equal(a, b) for a, b in zip(got, want))

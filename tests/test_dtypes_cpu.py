"""Layers of types that the library does not compute in are refused: their rows would be read as halves."""
import pytest

from helpers import pkg


@pytest.mark.parametrize("name", ["float32", "float64", "int16", "float8_e4m3fn"])
def test_other_types_are_refused(name):
    import torch

    p, dtype = pkg(), getattr(torch, name)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        p.LinearAttention(4, 4, 128, torch.zeros(4), 2, dtype=dtype, device="cpu")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        p.KvarnLayer(128, 4, 8, 4, torch.arange(4, dtype=torch.int32), dtype=dtype, device="cpu")


def test_both_types_are_taken():
    import torch

    p = pkg()
    for dtype, code in ((torch.float16, p.capi.DTYPE_F16), (torch.bfloat16, p.capi.DTYPE_BF16)):
        assert p.LinearAttention(4, 4, 128, torch.zeros(4), 2, dtype=dtype, device="cpu").c.dtype == code
        assert p.KvarnLayer(128, 4, 8, 4, torch.arange(4, dtype=torch.int32), dtype=dtype, device="cpu").c.dtype == code

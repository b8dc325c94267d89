"""Rotary positions: frequencies of the usual scalings for long contexts, and the turn of rows (kvb_rope_rows).  The append that turns keys on
the way is KvarnLayer.rope_append."""
from __future__ import annotations

import ctypes as C

import torch

from . import capi
from .cache import _DTYPE_CODES, check_indices, row_stride, stream_for

_SCALINGS = {"none": capi.ROPE_PLAIN, "linear": capi.ROPE_LINEAR, "ntk": capi.ROPE_NTK, "yarn": capi.ROPE_YARN}


class Rope:
    """The angles per position of a head's first `rotary_dim` dims, in device memory.  `scaling`: "none", "linear", "ntk" or "yarn", by `factor`
    ("yarn" also wants `original`, the length the model was trained at)."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original: int = 0, interleaved: bool = False,
                 device: str = "cuda"):
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling {scaling!r}: one of {', '.join(_SCALINGS)}")
        host, attention = (C.c_double * max(1, rotary_dim // 2))(), C.c_float()
        capi.check(capi.load().kvb_rope_frequencies(rotary_dim, base, _SCALINGS[scaling], factor, original, host, C.byref(attention)))
        self.rotary_dim, self.factor, self.interleaved = rotary_dim, attention.value, interleaved
        self.inv_freq = torch.tensor(list(host), dtype=torch.float64).to(device)
        self.c = capi.kvb_rope(inv_freq=self.inv_freq.data_ptr(), factor=self.factor, rotary_dim=rotary_dim, interleaved=int(interleaved))
        self.ref = C.byref(self.c)
        self.index = self.inv_freq.get_device()

    def rows(self, x: torch.Tensor, positions: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """x: [tokens, heads, head_dim] (fp16 or bf16), packed or part of wider rows; positions: int32 [tokens] on the device.  `out` may be x."""
        dtype = _DTYPE_CODES.get(x.dtype)
        if dtype is None or x.dim() != 3:
            raise ValueError(f"x: rows [tokens, heads, head_dim] of float16 or bfloat16, got {tuple(x.shape)} of {x.dtype}")
        tokens, heads, dim = x.shape
        at = check_indices(positions, tokens, "positions")
        stride = row_stride(x, heads, dim, x.dtype, tokens)
        out = torch.empty_like(x) if out is None else out
        capi.check(capi.load().kvb_rope_rows(self.ref, x.data_ptr(), stride, out.data_ptr(), row_stride(out, heads, dim, x.dtype, tokens), at, tokens, heads,
                                             dim, dtype, stream_for(self.index, x, positions, out)))
        return out

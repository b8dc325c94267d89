"""Linear attention with one decay for each head, the same at every token: layers of a hybrid model that keep a state per sequence instead of a cache."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import capi
from .cache import check_indices, dtype_code, row_stride, stream_for


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device, tokens, batch, v_heads, head_dim):
    return capi.load().kvb_linear_workspace_bytes(tokens, batch, v_heads, head_dim)


class LinearAttention:
    """One layer: the decay of its heads and a pool of states, [slots, v_heads, head_dim of k, head_dim of v] in fp32, zeros at first."""

    def __init__(self, qk_heads: int, v_heads: int, head_dim: int, log_decay: torch.Tensor, slots: int, dtype: torch.dtype = torch.bfloat16,
                 device: str = "cuda"):
        if tuple(log_decay.shape) != (v_heads,):
            raise ValueError(f"log_decay: [{v_heads}], got {tuple(log_decay.shape)}")
        code = dtype_code(dtype)
        self.qk_heads, self.v_heads, self.head_dim, self.slots, self.dtype = qk_heads, v_heads, head_dim, slots, dtype
        self.device = torch.device(device)
        self.state = torch.zeros((slots, v_heads, head_dim, head_dim), dtype=torch.float32, device=self.device)
        self.log_decay = log_decay.to(device=self.device, dtype=torch.float32).contiguous()
        self.error_word = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.c = capi.kvb_linear(state=self.state.data_ptr(), log_decay=self.log_decay.data_ptr(), slots=slots, qk_heads=qk_heads, v_heads=v_heads,
                                 head_dim=head_dim, dtype=code, error_word=self.error_word.data_ptr())
        self.ref = C.byref(self.c)
        self.index = self.state.get_device()
        self._ws = []

    def _device_key(self) -> int:
        return torch._C._cuda_getDevice() if self.device.type == "cuda" else -1

    def _out(self, tokens, v, out):
        if out is None:
            return torch.empty((tokens, self.v_heads, self.head_dim), dtype=self.dtype, device=v.device) if not v.is_contiguous() else torch.empty_like(v)
        if out.shape != (tokens, self.v_heads, self.head_dim) or out.dtype is not self.dtype or not out.is_contiguous():
            raise ValueError(f"out: packed rows [{tokens}, {self.v_heads}, {self.head_dim}] of {self.dtype}")
        return out

    def decode(self, q, k, v, scale: float, reads: torch.Tensor, writes: torch.Tensor, out=None) -> torch.Tensor:
        """One token of each sequence: q, k [batch, qk_heads, head_dim], v [batch, v_heads, head_dim]; reads, writes: int32 [batch] on the device, the
        slots a sequence's state is read from and written to (the same one for a step in place)."""
        batch, qk, d, dtype = q.shape[0], self.qk_heads, self.head_dim, self.dtype
        qs, ks, vs = row_stride(q, qk, d, dtype, batch), row_stride(k, qk, d, dtype, batch), row_stride(v, self.v_heads, d, dtype, batch)
        out = self._out(batch, v, out)
        capi.check(capi.load().kvb_linear_decode(self.ref, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, batch, check_indices(reads, batch, "reads"),
                                                 check_indices(writes, batch, "writes"), scale, out.data_ptr(), stream_for(self.index, q, k, v, reads, writes, out)))
        return out

    def workspace(self, tokens: int, batch: int) -> torch.Tensor:
        """Scratch for chunk calls: the layer's own, which its calls share, so they do not overlap on the GPU.  Where a call wants more, the next buffer is
        at least twice as large and the ones before stay as they are: a CUDA graph may have captured their addresses."""
        n = (_workspace_bytes(self._device_key(), tokens, batch, self.v_heads, self.head_dim) + 3) // 4
        if not self._ws or self._ws[-1].numel() < n:
            self._ws.append(torch.empty(max(n, 2 * self._ws[-1].numel()) if self._ws else n, dtype=torch.float32, device=self.device))
        return self._ws[-1]

    def chunk(self, q, k, v, offsets: torch.Tensor, scale: float, reads: torch.Tensor, writes: torch.Tensor, out=None) -> torch.Tensor:
        """Several tokens of each sequence, packed: rows offsets[b] .. offsets[b + 1] - 1 are sequence b's; offsets: int32 [batch + 1] on the device."""
        tokens, qk, d, dtype, batch = q.shape[0], self.qk_heads, self.head_dim, self.dtype, reads.shape[0]
        qs, ks, vs = row_stride(q, qk, d, dtype, tokens), row_stride(k, qk, d, dtype, tokens), row_stride(v, self.v_heads, d, dtype, tokens)
        out = self._out(tokens, v, out)
        stream = stream_for(self.index, q, k, v, offsets, reads, writes, out)
        capi.check(capi.load().kvb_linear_chunk(self.ref, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, check_indices(offsets, batch + 1, "offsets"),
                                                batch, tokens, check_indices(reads, batch, "reads"), check_indices(writes, batch, "writes"), scale,
                                                self.workspace(tokens, batch).data_ptr(), out.data_ptr(), stream))
        return out

    def errors(self) -> int:
        return int(self.error_word.item())

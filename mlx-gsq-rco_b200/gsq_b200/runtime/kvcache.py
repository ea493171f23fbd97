"""Quantised key/value cache of one attention layer.

Extends the reference, which keeps mlx_lm's fp16 cache.  The cache is four
plain tensors: one-byte codes ``k``, ``v`` [batch, heads, length, dim]
(``torch.int8`` or ``torch.float8_e4m3fn``) and fp32 scales ``k_scale``,
``v_scale`` [batch, heads, length], one per token and head; a stored vector is
``code * scale``.  ``kernels.kv_append`` writes it, ``kernels.kv_read`` reads
it back, ``kernels.cached_attention`` attends over it.
"""
from __future__ import annotations

import ctypes

import torch

KV_FORMATS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}  # by gsq_kv_format: 0, 1
_CODE = {torch.int8: 0, torch.float8_e4m3fn: 1}


class QuantizedKVCache:
    """A handle on the four tensors (not copied; all contiguous, on one CUDA device)."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "batch", "heads", "length", "dim", "fmt", "device", "pointers", "checked")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dim() != 4 or k.shape[3] not in (128, 256):
            raise ValueError("cache codes are [batch, heads, length, dim] with dim 128 or 256")
        if k.dtype not in _CODE or v.dtype != k.dtype:
            raise TypeError(f"cache codes must both be int8 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
        if v.shape != k.shape or k_scale.shape != k.shape[:3] or v_scale.shape != k.shape[:3]:
            raise ValueError("cache codes and scales must have matching shapes")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise TypeError("cache scales must be float32")
        tensors = (k, v, k_scale, v_scale)
        if any(t.device != k.device for t in tensors):
            raise RuntimeError("tensors on different devices")
        if k.device.type != "cuda":
            raise RuntimeError("gsq_b200 runs on CUDA tensors only (no CPU fallback)")
        if not all(t.is_contiguous() for t in tensors):
            raise ValueError("cache tensors must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = tensors
        self.batch, self.heads, self.length, self.dim = k.shape
        self.fmt, self.device = _CODE[k.dtype], k.device
        self.pointers = tuple(ctypes.c_void_p(t.data_ptr()) for t in tensors)
        self.checked: dict[tuple, tuple] = {}  # shapes and strides of calls seen, with what the C ABI takes for them

    def remember(self, key: tuple, call: tuple) -> tuple:
        """Keeps what was derived from a call's shapes, strides and types (never from its data or addresses)."""
        if len(self.checked) >= 1024:
            self.checked.clear()
        self.checked[key] = call
        return call

    @classmethod
    def empty(cls, batch: int, heads: int, length: int, dim: int, fmt: str = "int8", device="cuda") -> QuantizedKVCache:
        """A cache of zeros: ``fmt`` "int8" or "fp8"."""
        if fmt not in KV_FORMATS:
            raise NotImplementedError(f"no cache format {fmt!r}")
        shape = (batch, heads, length, dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(KV_FORMATS[fmt]) for _ in range(2)]
        return cls(*codes, *(torch.zeros(shape[:3], device=device) for _ in range(2)))

    @property
    def nbytes(self) -> int:
        return 2 * self.k.numel() + 8 * self.k_scale.numel()

    def sequences(self, count: int) -> QuantizedKVCache:
        """A handle on the first ``count`` sequences of the same tensors."""
        return QuantizedKVCache(self.k[:count], self.v[:count], self.k_scale[:count], self.v_scale[:count])

    def copy_sequence(self, source: int, targets: slice, length: int) -> None:
        """The first ``length`` positions of sequence ``source`` into the sequences ``targets``."""
        for t in (self.k.view(torch.int8), self.v.view(torch.int8), self.k_scale, self.v_scale):
            t[targets, :, :length].copy_(t[source:source + 1, :, :length].expand_as(t[targets, :, :length]))

"""Quantised key/value cache: writing, and reading back (csrc/kvcache.cu).

Extends the reference, which keeps an fp16 cache.  The format is in
``include/gsq_model.h`` (``gsq_kv_append``) and ``runtime/kvcache.py``.
"""
from __future__ import annotations

import ctypes

import torch

from ... import _lib

Strides = ctypes.c_int64 * 3
_I, _I64 = ctypes.c_int, ctypes.c_int64  # arguments in the C ABI's own types are not converted again at each call


def check_start(start: torch.Tensor, batch: int, device) -> int:
    """The stride of ``start``: int32, one position per sequence or one for all."""
    if start.dtype != torch.int32:
        raise TypeError(f"start must be int32, got {start.dtype}")
    if start.device != device:
        raise RuntimeError("tensors on different devices")
    if start.dim() != 1 or start.shape[0] not in (1, batch):
        raise ValueError(f"start must hold 1 or {batch} positions")
    return 0 if start.shape[0] == 1 else start.stride(0)


def check_counts(counts: torch.Tensor | None, batch: int, device) -> int | None:
    """The address of ``counts``: int32, one per sequence; None without it."""
    if counts is None:
        return None
    if counts.dtype != torch.int32:
        raise TypeError(f"counts must be int32, got {counts.dtype}")
    if counts.device != device:
        raise RuntimeError("tensors on different devices")
    if counts.shape != (batch,) or not counts.is_contiguous():
        raise ValueError(f"counts must hold {batch} contiguous values")
    return counts.data_ptr()


def kv_append(cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
              counts: torch.Tensor | None = None) -> None:
    """Quantises the new keys and values ``k``, ``v`` [batch, tokens, heads,
    dim] (fp32, fp16 or bf16; the last dimension contiguous, any other
    strides) into ``cache`` at positions ``start[b]``, ``start[b] + 1``, ...

    ``start``: int32 on the device, one position per sequence or one for all;
    ``counts``: int32, sequence b has only ``counts[b]`` new tokens and the
    rest of its rows is padding.  A position outside the cache is not written
    and shows as 3 in ``_lib.device_status``."""
    key = ("append", k.shape, v.shape, k.stride(), v.stride(), k.dtype, v.dtype)
    call = cache.checked.get(key)
    if call is None:
        if k.shape != v.shape or k.dim() != 4 or k.shape[0] != cache.batch or k.shape[2:] != (cache.heads, cache.dim):
            raise ValueError(f"expected k and v [{cache.batch}, tokens, {cache.heads}, {cache.dim}], "
                             f"got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.dtype not in _lib.DTYPE_CODES or v.dtype != k.dtype:
            raise TypeError(f"unsupported key/value dtypes {k.dtype}, {v.dtype}")
        if k.stride(3) != 1 or v.stride(3) != 1:
            return kv_append(cache, k.contiguous(), v.contiguous(), start, counts)
        call = cache.remember(key, (_I(_lib.DTYPE_CODES[k.dtype]), _I64(cache.batch), _I64(k.shape[1]),
                                    _I64(cache.heads), _I64(cache.dim), Strides(*k.stride()[:3]),
                                    Strides(*v.stride()[:3])))
    dev = cache.device
    if k.device != dev or v.device != dev:
        raise RuntimeError("tensors on different devices")
    stride = check_start(start, cache.batch, dev)
    _lib.launch(dev, _lib.load().gsq_kv_append, k.data_ptr(), v.data_ptr(), *call, start.data_ptr(), stride,
                None if counts is None else check_counts(counts, cache.batch, dev), cache.fmt, *cache.pointers,
                cache.length)


def kv_read(cache, start: torch.Tensor, tokens: int, *, counts: torch.Tensor | None = None,
            dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """Reads positions ``start[b]`` .. ``start[b] + tokens - 1`` of every
    sequence back as (k, v) [batch, tokens, heads, dim] of ``dtype``: code *
    scale in fp32, rounded once.  Padding (``counts``) and positions outside
    the cache read as zeros."""
    if dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"unsupported output dtype {dtype}")
    if tokens < 0:
        raise ValueError("negative token count")
    dev = cache.device
    stride = check_start(start, cache.batch, dev)
    k = torch.empty((cache.batch, tokens, cache.heads, cache.dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _lib.launch(dev, _lib.load().gsq_kv_read, cache.fmt, *cache.pointers, cache.batch, cache.heads, cache.length,
                cache.dim, start.data_ptr(), stride,
                None if counts is None else check_counts(counts, cache.batch, dev), tokens, k.data_ptr(),
                v.data_ptr(), _lib.DTYPE_CODES[dtype])
    return k, v

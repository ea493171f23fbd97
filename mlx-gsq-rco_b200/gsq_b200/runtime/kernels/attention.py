"""Attention of new tokens over the quantised cache (csrc/cached_attn.cu).

Extends the reference, whose attention is mlx_lm's over an fp16 cache.  One
entry point for single tokens, chunks of a prompt and trees of drafted
tokens; the formula is in ``include/gsq_model.h`` (``gsq_cached_attention``).
"""
from __future__ import annotations

import numpy as np
import torch

from ... import _lib
from .kvcache import _I, _I64, Strides, check_counts, check_start


def tree_mask(parents, device="cuda") -> torch.Tensor:
    """The mask of a drafted tree for ``cached_attention``: int32 words
    [n, ceil(n / 32)] (or [batch, n, ...] for a list of trees of equal size),
    bit j of row i set where token j is token i or an ancestor of it.
    ``parents[i]`` is the index of token i's parent, below i, or -1 where it
    follows the cached text directly."""
    p = np.asarray(parents.cpu() if isinstance(parents, torch.Tensor) else parents, dtype=np.int64)
    if p.ndim == 2:
        return torch.stack([tree_mask(row, device) for row in p]) if len(p) else \
            torch.empty((0, p.shape[1], (p.shape[1] + 31) // 32), dtype=torch.int32, device=device)
    if p.ndim != 1:
        raise ValueError("parents must be [n] or [batch, n]")
    n = len(p)
    if ((p < -1) | (p >= np.arange(n))).any():
        raise ValueError("every parent comes before its children (-1: the cached text)")
    bits = np.zeros((n, (n + 31) // 32 * 32), dtype=np.uint8)
    for i in range(n):
        if p[i] >= 0:
            bits[i] = bits[p[i]]
        bits[i, i] = 1
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view("<i4").copy()).to(device)


def cached_attention(q: torch.Tensor, cache, start: torch.Tensor, *, counts: torch.Tensor | None = None,
                     tree: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v [* sigmoid(gate)] of the new tokens' queries
    ``q`` [batch, n, heads, dim] (fp16 or bf16) over ``cache``, which holds
    their keys and values already (``kv_append`` with the same ``start`` and
    ``counts``); q's heads are a multiple of the cache's.

    Token i of sequence b sees positions 0 .. start[b] + i, or with ``tree``
    (int32 words [n, ceil(n / 32)] or [batch, n, ceil(n / 32)], see
    ``tree_mask``; n up to 1024) positions below start[b] and the new tokens
    whose bit is set in its row.  Rows that see nothing, and padding (i >=
    counts[b]), give zeros.  ``gate``: fp32 of q's shape, any strides with
    the last dimension contiguous; ``scale``: dim ** -0.5 by default.
    Returns [batch, n, heads, dim] in q's dtype (``out``, when given)."""
    lib = _lib.load()
    key = ("attend", q.shape, q.stride(), q.dtype)
    call = cache.checked.get(key)
    if call is None:
        call = _check_queries(q, cache, key)
    direct, need, words, args = call
    dev = cache.device
    batch, n = q.shape[:2]
    if q.device != dev:
        raise RuntimeError("tensors on different devices")
    stride = check_start(start, batch, dev)
    if not direct or q.data_ptr() % 16:  # the kernels read rows of q with 16-byte loads
        return cached_attention(torch.empty(q.shape, dtype=q.dtype, device=dev).copy_(q), cache, start, counts=counts,
                                tree=tree, gate=gate, scale=scale, out=out)
    tree_ptr, tree_stride = None, 0
    if tree is not None:
        if tree.dtype != torch.int32:
            raise TypeError(f"a tree mask is int32 words, got {tree.dtype}")
        if tree.shape not in ((n, words), (batch, n, words)) or n > 1024:
            raise ValueError(f"expected a tree mask [{n}, {words}] or [{batch}, {n}, {words}] with n at most 1024, "
                             f"got {tuple(tree.shape)}")
        if tree.device != dev:
            raise RuntimeError("tensors on different devices")
        tree = tree.contiguous()
        tree_ptr, tree_stride = tree.data_ptr(), n * words if tree.dim() == 3 else 0
    gate_ptr, gate_strides = None, None
    if gate is not None:
        if gate.dtype != torch.float32 or gate.shape != q.shape:
            raise ValueError(f"the gate must be float32 of q's shape {tuple(q.shape)}")
        if gate.device != dev:
            raise RuntimeError("tensors on different devices")
        gs = gate.stride()
        if gs[3] != 1:
            gate = gate.contiguous()
            gs = gate.stride()
        gate_ptr, gate_strides = gate.data_ptr(), Strides(*gs[:3])
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous() or \
            out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of q's shape, dtype and device")
    # this call's alone, held until its launches are queued: from then on the stream orders the memory's next use
    ws = q.new_empty(need // 2) if need else None
    _lib.launch(dev, lib.gsq_cached_attention, q.data_ptr(), *args, *cache.pointers, cache.length, start.data_ptr(),
                stride, None if counts is None else check_counts(counts, batch, dev), tree_ptr, tree_stride, gate_ptr,
                gate_strides, cache.dim ** -0.5 if scale is None else float(scale), out.data_ptr(),
                None if ws is None else ws.data_ptr(), need)
    return out


def _check_queries(q: torch.Tensor, cache, key: tuple) -> tuple:
    """(whether the kernels read q as it is, workspace bytes, words of a tree's row, C arguments) for q's shape."""
    if q.dim() != 4 or q.shape[0] != cache.batch or q.shape[3] != cache.dim:
        raise ValueError(f"expected q [{cache.batch}, n, heads, {cache.dim}], got {tuple(q.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"queries must be float16 or bfloat16, got {q.dtype}")
    batch, n, heads, dim = q.shape
    if heads == 0 or heads % cache.heads:
        raise ValueError(f"{heads} query heads are not a multiple of the cache's {cache.heads}")
    s = q.stride()
    need = _lib.load().gsq_cached_attention_workspace_size(batch, n, heads, cache.heads, dim, cache.length)
    args = (_I(_lib.DTYPE_CODES[q.dtype]), Strides(*s[:3]), _I64(batch), _I64(n), _I64(heads), _I64(cache.heads),
            _I64(dim), _I(cache.fmt))
    return cache.remember(key, (s[3] == 1 and not (s[0] | s[1] | s[2]) % 8, need, (n + 31) // 32, args))

"""Penalties, biases and masks on logits, and the token they lead to
(csrc/logits.cu).

The reference has no sampler of its own (it hands logits to mlx_lm).  The
order of the steps is in ``include/gsq_model.h`` (``gsq_adjust_logits``).
"""
from __future__ import annotations

import torch

from ... import _lib


def _per_row(t: torch.Tensor, name: str, rows: int, dev) -> int:
    if t.dtype != torch.float32 or t.shape != (rows,) or t.device != dev or t.stride(0) != 1:
        raise ValueError(f"{name} must be {rows} contiguous float32 values on {dev}")
    return t.data_ptr()


def adjust_logits(logits: torch.Tensor, *, history=None, repetition: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  record: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The adjusted fp32 rows of ``logits`` [rows, vocab] (fp32, fp16 or bf16)
    and each row's token of the highest value (int32 [rows]; the lowest of
    equal ones).

    For the tokens that ``history`` (a ``TokenHistory``, row r for row r) has
    seen: divided (positive) or multiplied by ``repetition``; for those of its
    output also minus ``frequency`` * count and ``presence`` (each fp32
    [rows]).  Then plus ``bias_values`` at ``bias_ids`` ([rows, up to 65536];
    int32; ids outside the vocabulary are padding, repeated ids add up), then
    -inf where ``allowed`` (int32 words [rows, ceil(vocab / 32)], or [ceil(vocab
    / 32)] for all rows) has no bit.  ``out`` may be ``logits`` itself when it
    is contiguous fp32.  With ``record`` the history learns the tokens."""
    if logits.dim() != 2 or not 0 < logits.shape[1] <= 1 << 20:
        raise ValueError(f"expected logits [rows, vocab] with vocab at most 2^20, got {tuple(logits.shape)}")
    if logits.dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"unsupported logits dtype {logits.dtype}")
    dev = logits.device
    if dev.type != "cuda":
        raise RuntimeError("gsq_b200 runs on CUDA tensors only (no CPU fallback)")
    rows, vocab = logits.shape
    words = (vocab + 31) // 32
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    seen_ptr = counts_ptr = None
    if history is not None:
        if history.vocab != vocab or history.rows < rows:
            raise ValueError(f"a history of {history.rows} rows and {history.vocab} tokens does not fit "
                             f"logits {tuple(logits.shape)}")
        if history.device != dev:
            raise RuntimeError("tensors on different devices")
        seen_ptr, counts_ptr = history.seen.data_ptr(), history.counts.data_ptr()
    elif record or repetition is not None or frequency is not None or presence is not None:
        raise ValueError("penalties and recording need a history")
    biases = 0
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values come together")
    if bias_ids is not None:
        if bias_ids.dtype != torch.int32 or bias_values.dtype != torch.float32:
            raise TypeError("bias_ids must be int32 and bias_values float32")
        if bias_ids.dim() != 2 or bias_ids.shape[0] != rows or bias_values.shape != bias_ids.shape or \
                bias_ids.shape[1] > 65536:
            raise ValueError(f"expected bias_ids and bias_values [{rows}, up to 65536]")
        if bias_ids.device != dev or bias_values.device != dev:
            raise RuntimeError("tensors on different devices")
        bias_ids, bias_values = bias_ids.contiguous(), bias_values.contiguous()
        biases = bias_ids.shape[1]
    allowed_ptr, allowed_stride = None, 0
    if allowed is not None:
        if allowed.dtype != torch.int32:
            raise TypeError(f"allowed is int32 words, got {allowed.dtype}")
        if allowed.shape not in ((words,), (rows, words)):
            raise ValueError(f"expected allowed [{words}] or [{rows}, {words}], got {tuple(allowed.shape)}")
        if allowed.device != dev:
            raise RuntimeError("tensors on different devices")
        allowed = allowed.contiguous()
        allowed_ptr, allowed_stride = allowed.data_ptr(), words if allowed.dim() == 2 else 0
    if out is None:
        out = logits.new_empty((rows, vocab), dtype=torch.float32)
    elif out.shape != (rows, vocab) or out.dtype != torch.float32 or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous float32 tensor of the logits' shape and device")
    nxt = logits.new_empty(rows, dtype=torch.int32)
    _lib.launch(dev, _lib.load().gsq_adjust_logits, logits.data_ptr(), _lib.DTYPE_CODES[logits.dtype],
                max(logits.stride(0), vocab), rows, vocab, seen_ptr, counts_ptr,
                None if repetition is None else _per_row(repetition, "repetition", rows, dev),
                None if frequency is None else _per_row(frequency, "frequency", rows, dev),
                None if presence is None else _per_row(presence, "presence", rows, dev),
                bias_ids.data_ptr() if biases else None, bias_values.data_ptr() if biases else None, biases, allowed_ptr,
                allowed_stride, out.data_ptr(), nxt.data_ptr(), int(record))
    return out, nxt


def record_tokens(history, tokens: torch.Tensor, *, generated: bool = True) -> None:
    """Row r of ``history`` learns ``tokens[r]`` (int32 [rows, n], rows up to
    the history's; tokens outside the vocabulary are padding): as output, or
    with ``generated=False`` as prompt (seen, not counted)."""
    if tokens.dtype != torch.int32:
        raise TypeError(f"tokens must be int32, got {tokens.dtype}")
    if tokens.dim() != 2 or tokens.shape[0] > history.rows:
        raise ValueError(f"expected tokens [up to {history.rows}, n], got {tuple(tokens.shape)}")
    dev = history.device
    if tokens.device != dev:
        raise RuntimeError("tensors on different devices")
    tokens = tokens.contiguous()
    _lib.launch(dev, _lib.load().gsq_record_tokens, tokens.data_ptr(), tokens.shape[1], tokens.shape[0],
                tokens.shape[1], history.vocab, history.seen.data_ptr(), history.counts.data_ptr(), int(generated))

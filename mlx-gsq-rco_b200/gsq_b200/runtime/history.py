"""What each row of logits has seen: the tokens behind repetition, frequency
and presence penalties, kept on the device so that a captured decode graph
can go on with them."""
from __future__ import annotations

import torch


class TokenHistory:
    """``seen``: int32 words [rows, ceil(vocab / 32)], bit v % 32 of word
    v // 32 set for every token v of the row's prompt or output; ``counts``:
    int32 [rows, vocab], how often the row's output holds each token (zero
    wherever the bit is not set).  The tensors are held, not copied."""

    __slots__ = ("seen", "counts", "rows", "vocab", "device")

    def __init__(self, seen: torch.Tensor, counts: torch.Tensor):
        if counts.dim() != 2 or seen.shape != (counts.shape[0], (counts.shape[1] + 31) // 32):
            raise ValueError("a history is seen [rows, ceil(vocab / 32)] and counts [rows, vocab]")
        if seen.dtype != torch.int32 or counts.dtype != torch.int32:
            raise TypeError("seen and counts must be int32")
        if seen.device != counts.device:
            raise RuntimeError("tensors on different devices")
        if counts.device.type != "cuda":
            raise RuntimeError("gsq_b200 runs on CUDA tensors only (no CPU fallback)")
        if not (seen.is_contiguous() and counts.is_contiguous()):
            raise ValueError("seen and counts must be contiguous")
        self.seen, self.counts, self.device = seen, counts, counts.device
        self.rows, self.vocab = counts.shape

    @classmethod
    def empty(cls, rows: int, vocab: int, device="cuda") -> TokenHistory:
        return cls(torch.zeros(rows, (vocab + 31) // 32, dtype=torch.int32, device=device),
                   torch.zeros(rows, vocab, dtype=torch.int32, device=device))

    def clear(self) -> None:
        self.seen.zero_()
        self.counts.zero_()

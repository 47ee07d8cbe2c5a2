"""Per-request controls on next-token logits, between the lm_head and the
sampler (``nova_b200.sampling``): penalties for repeated tokens, token biases
and grammar masks, in one pass over the logits.

    history = new_history(rows, vocab)                    # per request: what it has seen
    add_prompt(history, prompt_ids, offsets)
    ...
    x = adjust_logits(logits, history=history, repetition=..., frequency=..., presence=...,
                      bias=LogitBias([{42: -100.0}, {}], vocab), allowed=masks, allowed_row=which)
    tok = sample_topk(x, temperature=..., top_k=..., uniform=...)
    add_generated(history, tok)

The repetition rule is that of the reference's ``sample_next`` (src/chat.py:58-61).
"""

from __future__ import annotations

from typing import Mapping, Sequence

import numpy as np
import torch

from . import _lib

CHUNK = 2048     # tokens per bias list: NOVA_LOGITS_CHUNK of include/nova_b200.h


class LogitBias:
    """Additive biases of each row: ``entries[row]`` maps token numbers to fp32
    values.  Built once per change on the host, kept on the device."""

    def __init__(self, entries: Sequence[Mapping[int, float]], vocab: int, device: torch.device | str = "cuda") -> None:
        self.rows, self.vocab = len(entries), int(vocab)
        chunks = -(-self.vocab // CHUNK)
        counts = np.fromiter((len(e) for e in entries), dtype=np.int64, count=len(entries))
        n = int(counts.sum())
        token = np.fromiter((t for e in entries for t in e), dtype=np.int64, count=n)
        value = np.fromiter((v for e in entries for v in e.values()), dtype=np.float32, count=n)
        if n and (token.min() < 0 or token.max() >= self.vocab):
            raise ValueError(f"bias tokens must lie in [0, {self.vocab})")
        row = np.repeat(np.arange(self.rows), counts)
        bucket = row * chunks + token // CHUNK
        order = np.argsort(bucket, kind="stable")
        off = np.zeros(self.rows * chunks + 1, dtype=np.int64)
        np.cumsum(np.bincount(bucket, minlength=self.rows * chunks), out=off[1:])
        # offsets, tokens and value bits in one copy
        packed = np.concatenate([off.astype(np.int32), token[order].astype(np.int32), value[order].view(np.int32)])
        self.buffer = torch.from_numpy(packed).to(device)
        m = len(off)
        self.off, self.token = self.buffer[:m], self.buffer[m:m + n]
        self.value = self.buffer[m + n:].view(torch.float32)
        own = _lib.stream_of(self.buffer.device) if self.buffer.is_cuda else 0
        self._handle = (self.rows, self.vocab, n, own, self.buffer)      # what csrc/binding.cpp reads


def new_history(rows: int, vocab: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """Empty history, int16 ``[rows, vocab]``: low 15 bits count how often a token
    was generated, the top bit says that it is in the prompt."""
    return torch.zeros(rows, vocab, dtype=torch.int16, device=device)


def _check_history(history: torch.Tensor) -> None:
    if not history.is_cuda or history.dtype != torch.int16 or history.dim() != 2 or history.stride(1) != 1:
        raise ValueError("history must be CUDA int16 [rows, vocab] with a contiguous last dimension")


def _history_add(history: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor | None, prompt: bool) -> None:
    _check_history(history)
    rows, vocab = history.shape
    if tokens.dtype != torch.int64 or tokens.device != history.device or not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous int64 on the history's device")
    if offsets is None:
        if tokens.numel() != rows:
            raise ValueError(f"one token per row ({rows}) is needed without offsets, got {tokens.numel()}")
    elif (offsets.dtype != torch.int32 or tuple(offsets.shape) != (rows + 1,) or offsets.device != history.device
          or not offsets.is_contiguous()):
        raise ValueError(f"offsets must be contiguous int32 [{rows + 1}] on the history's device")
    with torch.cuda.device(history.device):       # the launch goes to the current device
        _lib.call("nova_history_add", history.data_ptr(), history.stride(0), tokens.data_ptr(), _lib.ptr(offsets),
                  tokens.numel(), rows, vocab, int(prompt), _lib.stream_of(history.device))


def add_prompt(history: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """Enter prompt tokens: int64, row r's are ``tokens[offsets[r]:offsets[r + 1]]``
    (int32 offsets on the device; without them one token per row).  Tokens
    outside the vocabulary and offsets outside the tokens are skipped."""
    _history_add(history, tokens, offsets, True)


def add_generated(history: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """Count generated tokens, as :func:`add_prompt` (e.g. the sampler's result)."""
    _history_add(history, tokens, offsets, False)


def adjust_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                  repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, bias: LogitBias | None = None,
                  allowed: torch.Tensor | None = None, allowed_row: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits fp16 or fp32 ``[rows, vocab]`` under each row's controls (one launch).

    ``repetition`` / ``frequency`` / ``presence``: fp32 ``[rows]``, applied where
    ``history`` (:func:`new_history`) has the token; ``bias``: added after them;
    ``allowed``: int32 ``[masks, ceil(vocab / 32)]`` bit masks (bit t % 32 of word
    t // 32), ``allowed_row`` int32 ``[rows]`` the mask of each row (negative:
    none; default: row i has mask i).  What a mask forbids becomes -inf whatever
    it was, NaN included; a row whose mask leaves nothing is all -inf.  ``out``
    may be ``logits``.  Returns a tensor of the logits' type."""
    return _lib.fast().adjust_logits(logits, history, repetition, frequency, presence,
                                     None if bias is None else bias._handle, allowed, allowed_row, out)

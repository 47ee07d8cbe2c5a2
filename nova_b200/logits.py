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

CHUNK = 2048     # tokens per bias list (one CTA's tokens)
_ADJUST = _lib.Entry("nova_adjust_logits", _lib.LogitsArgs, _lib._P)


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
        at = self.buffer.data_ptr()
        self._pointers = (at, at + 4 * m, at + 4 * (m + n)) if n else (0, 0, 0)


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
    _lib.call("nova_history_add", history.data_ptr(), history.stride(0), tokens.data_ptr(), _lib.ptr(offsets),
              tokens.numel(), rows, vocab, int(prompt), _lib.stream_of(history.device))


def add_prompt(history: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """Enter prompt tokens: int64, row r's are ``tokens[offsets[r]:offsets[r + 1]]``
    (int32 offsets on the device; without them one token per row).  Tokens
    outside the vocabulary are skipped."""
    _history_add(history, tokens, offsets, True)


def add_generated(history: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """Count generated tokens, as :func:`add_prompt` (e.g. the sampler's result)."""
    _history_add(history, tokens, offsets, False)


def _control(t: torch.Tensor, name: str, rows: int, device: int, history: torch.Tensor | None) -> int:
    if t.dtype != torch.float32 or t.shape != (rows,) or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 [{rows}] on the logits' device")
    if history is None:
        raise ValueError(f"{name} needs a history")
    return t.data_ptr()


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
    i, dtype, shape = logits.get_device(), logits.dtype, logits.shape
    if i < 0 or len(shape) != 2 or (dtype != torch.float16 and dtype != torch.float32) or logits.stride(1) != 1:
        raise ValueError("logits must be CUDA float16 or float32 [rows, vocab] with a contiguous last dimension")
    rows, vocab = shape
    if out is None:
        out = torch.empty_strided(shape, (vocab, 1), dtype=dtype, device=logits.device)
    elif out.dtype != dtype or out.shape != shape or out.get_device() != i or out.stride(1) != 1:
        raise ValueError("out must have the shape, type and device of logits and a contiguous last dimension")
    hist = hist_stride = 0
    if history is not None:
        if history.dtype != torch.int16 or history.shape != shape or history.get_device() != i or history.stride(1) != 1:
            raise ValueError(f"history must be int16 {tuple(shape)} on the logits' device with a contiguous last dimension")
        hist, hist_stride = history.data_ptr(), history.stride(0)
    rep = freq = pres = 0
    if repetition is not None:
        rep = _control(repetition, "repetition", rows, i, history)
    if frequency is not None:
        freq = _control(frequency, "frequency", rows, i, history)
    if presence is not None:
        pres = _control(presence, "presence", rows, i, history)
    biases = (0, 0, 0)
    if bias is not None:
        if bias.rows != rows or bias.vocab != vocab or bias.buffer.get_device() != i:
            raise ValueError(f"bias is for [{bias.rows}, {bias.vocab}] logits, got {tuple(shape)}")
        biases = bias._pointers
    mask = masks = mask_stride = mask_row = 0
    if allowed is not None:
        words = (vocab + 31) // 32
        if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.get_device() != i:
            raise ValueError(f"allowed must be int32 [masks, {words}] on the logits' device")
        masks, width = allowed.shape
        mask_stride, last = allowed.stride()
        if masks < 1 or width < words or last != 1 or (masks > 1 and mask_stride < width):
            raise ValueError(f"allowed must be int32 [masks, {words}] with rows of their own, got {tuple(allowed.shape)}")
        mask, mask_stride = allowed.data_ptr(), max(mask_stride, width)
        if allowed_row is not None:
            if allowed_row.dtype != torch.int32 or allowed_row.shape != (rows,) or allowed_row.get_device() != i \
                    or not allowed_row.is_contiguous():
                raise ValueError(f"allowed_row must be contiguous int32 [{rows}] on the logits' device")
            mask_row = allowed_row.data_ptr()
        elif masks != rows:
            raise ValueError(f"{masks} masks for {rows} rows need allowed_row")
    elif allowed_row is not None:
        raise ValueError("allowed_row needs allowed")
    _ADJUST(_ADJUST.pack(logits.data_ptr(), logits.stride(0), dtype == torch.float32, out.data_ptr(), out.stride(0), hist,
                         hist_stride, rep, freq, pres, *biases, mask, masks, mask_stride, mask_row, rows, vocab),
            _lib.raw_stream(i))
    return out

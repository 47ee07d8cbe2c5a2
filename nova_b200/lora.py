"""Low-rank adapters of many requests at once, beside a projection whose weights
they share (the NF4 linears: ``nova_b200.kernels.nf4_gemm``).

    plan = LoraPlan(token_counts, adapter_of_request, ranks)       # once per step
    y = nf4_gemm(x, ...)                                           # the shared projection
    y = lora_add(x, y, a, b, plan, scaling=scaling, out=y)         # + s (x A^T) B^T per request

No counterpart in the reference.
"""

from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

from . import _lib

MAX_RANK = 128


class LoraPlan:
    """Which adapter each token row of a step takes.

    ``token_counts``: rows of each request, one after another; ``adapters``: the
    adapter of each request, negative for none; ``ranks``: rank of every adapter
    (1 .. 128; 0 switches one off).  Rows of one adapter are gathered into tiles
    whatever their requests; the plan serves every projection of the step.  It
    holds device buffers and is used by one stream at a time."""

    def __init__(self, token_counts: Sequence[int], adapters: Sequence[int], ranks: Sequence[int], *,
                 device: torch.device | str = "cuda") -> None:
        counts, which = np.asarray(token_counts, dtype=np.int64), np.asarray(adapters, dtype=np.int64)
        rank = np.asarray(ranks, dtype=np.int64)
        if counts.ndim != 1 or counts.shape != which.shape or rank.ndim != 1:
            raise ValueError("token_counts and adapters must be flat and of one length, ranks flat")
        if (counts < 0).any():
            raise ValueError("token_counts must not be negative")
        if len(which) and which.max() >= len(rank):
            raise ValueError(f"adapter {which.max()} of {len(rank)}")
        if len(rank) and (rank.min() < 0 or rank.max() > MAX_RANK):
            raise ValueError(f"ranks must lie in [0, {MAX_RANK}]")
        self.tokens, self.adapters = int(counts.sum()), len(rank)
        self.max_rank = int(rank.max()) if len(rank) else 0
        of_row = np.repeat(np.where(which < 0, -1, which), counts)
        if len(rank):
            of_row = np.where((of_row >= 0) & (rank[of_row] == 0), -1, of_row)
        rows = np.argsort(of_row, kind="stable")
        values, first, n = np.unique(of_row[rows], return_index=True, return_counts=True)
        busy = n[values >= 0]
        # 16-row tiles are one launch, 8 CTAs each; once they no longer fit the GPU at once (two CTAs on each of 148 SMs
        # are 37 tiles: about 40), 64-row tiles in two launches are faster if they are fewer: 300 rows of one adapter 14 us against 22, 700 rows 22.5
        # and 21, 2800 rows 56 and 38; one row of each of 64 adapters 21 us against 29
        small, large = (-(-busy // 16)).sum(), (-(-busy // 64)).sum()
        self.tile_rows = 64 if small > 40 and 2 * large <= small else 16
        # per tile: adapter, rank, rows, 0, then the rows, padded with -1
        rec = 4 + self.tile_rows
        counts = -(-n // self.tile_rows)
        self.n_tiles = int(counts.sum())
        tiles = np.full((self.n_tiles, rec), -1, dtype=np.int32)
        group = np.repeat(np.arange(len(values)), counts)                       # which adapter's rows
        nth = np.arange(self.n_tiles) - np.repeat(np.cumsum(counts) - counts, counts)
        tiles[:, 0] = values[group]
        tiles[:, 1] = np.where(values[group] >= 0, rank[values[group]] if len(rank) else 0, 0)
        tiles[:, 2] = np.minimum(self.tile_rows, n[group] - nth * self.tile_rows)
        tiles[:, 3] = 0
        start = first[group] + nth * self.tile_rows
        at = start[:, None] + np.arange(self.tile_rows)
        inside = np.arange(self.tile_rows) < tiles[:, 2:3]
        tiles[:, 4:][inside] = rows[at[inside]]
        self.device = torch.device(device)
        self.buffer = torch.from_numpy(tiles.reshape(-1)).to(self.device)
        need = _lib.ctypes.c_int64(0)
        _lib.call("nova_lora_workspace_bytes", self.n_tiles, self.tile_rows, self.max_rank, _lib.ctypes.byref(need))
        self.workspace = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._handle = 0                      # on the host: for inspection only
        if self.buffer.is_cuda:               # what csrc/binding.cpp reads (LoraHandle)
            self._fields = (_lib.ctypes.c_int64 * 10)(
                self.buffer.data_ptr(), self.workspace.data_ptr(), need.value, self.buffer.get_device(),
                _lib.stream_of(self.buffer.device), self.n_tiles, self.tile_rows, self.tokens, self.adapters, self.max_rank)
            self._handle = _lib.handle(self._fields, _lib.LORA_PLAN)

    def _on_other_stream(self) -> None:
        """A stream other than the plan's own uses its buffers: the allocator must know."""
        current = torch.cuda.current_stream(self.buffer.device)
        self.buffer.record_stream(current)
        self.workspace.record_stream(current)


def lora_add(x: torch.Tensor, base: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan, *,
             scaling: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``base + scaling[a] * (x A_a^T) B_a^T`` for every row's adapter ``a``: one
    launch, or two where the plan has 64-row tiles.

    ``x`` fp16 ``[tokens, K]``; ``base`` fp16 ``[tokens, N]`` (the shared
    projection's output); ``a`` fp16 ``[adapters, R, K]``; ``b`` fp16 ``[adapters,
    N, R]``, R a multiple of 8 up to 128 and at least every rank (entries past an
    adapter's rank are not read); ``scaling`` fp32 ``[adapters]``.  ``out`` may be
    ``base``; rows without an adapter are then left alone.  Returns fp16
    ``[tokens, N]``.  Between the products a row of ``x A_a^T`` is fp16 at a power
    of two of its own, so any size of ``x``, ``a`` and ``scaling`` keeps its 11 bits."""
    return _lib.fast().lora_add(x, base, a, b, plan, scaling, out)

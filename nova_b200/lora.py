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
_F16 = torch.float16
_ADD = _lib.Entry("nova_lora_add", _lib.LoraArgs, _lib._P)


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
        # 16-row tiles are one launch, 8 CTAs each; once they no longer fit the GPU at once (two CTAs per SM), 64-row
        # tiles in two launches are faster: 300 rows 14 us against 22, 700 rows 22.5 and 21, 2800 rows 56 and 38
        self.tile_rows = 64 if (-(-busy // 16)).sum() > 40 else 16
        tiles = []
        for v, f, m in zip(values.tolist(), first.tolist(), n.tolist()):
            r = int(rank[v]) if v >= 0 else 0
            tiles += [(v, r, f + i, min(self.tile_rows, m - i)) for i in range(0, m, self.tile_rows)]
        self.n_tiles = len(tiles)
        host = np.concatenate([np.asarray(tiles, dtype=np.int32).reshape(-1), rows.astype(np.int32)])
        self.device = torch.device(device)
        self.buffer = torch.from_numpy(host).to(self.device)
        self._index = self.buffer.get_device()
        self._stream = _lib.raw_stream(self._index) if self._index >= 0 else 0
        self._tiles = self.buffer.data_ptr()
        self._rows = self._tiles + 16 * self.n_tiles
        need = _lib.ctypes.c_int64(0)
        _lib.call("nova_lora_workspace_bytes", self.n_tiles, self.tile_rows, self.max_rank, _lib.ctypes.byref(need))
        self.workspace = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._workspace = (self.workspace.data_ptr(), need.value)

    def _current(self) -> int:
        """The current stream; tells the allocator when it is not the plan's own."""
        stream = _lib.raw_stream(self._index)
        if stream != self._stream:
            current = torch.cuda.current_stream(self._index)
            self.buffer.record_stream(current)
            self.workspace.record_stream(current)
        return stream


def lora_add(x: torch.Tensor, base: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan, *,
             scaling: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``base + scaling[a] * (x A_a^T) B_a^T`` for every row's adapter ``a``, one launch.

    ``x`` fp16 ``[tokens, K]``; ``base`` fp16 ``[tokens, N]`` (the shared
    projection's output); ``a`` fp16 ``[adapters, R, K]``; ``b`` fp16 ``[adapters,
    N, R]``, R a multiple of 8 up to 128 and at least every rank (entries past an
    adapter's rank are not read); ``scaling`` fp32 ``[adapters]``.  ``out`` may be
    ``base``; rows without an adapter are then left alone.  Returns fp16
    ``[tokens, N]``."""
    i = plan._index
    if i < 0:
        raise ValueError("the plan is not on a CUDA device")
    for t, name in ((x, "x"), (base, "base"), (a, "a"), (b, "b")):
        if t.dtype != _F16 or t.get_device() != i:
            raise ValueError(f"{name} must be float16 on the plan's CUDA device, got {t.dtype} on {t.device}")
    if x.dim() != 2 or base.dim() != 2 or a.dim() != 3:
        raise ValueError("x and base must be 2-D, a and b 3-D")
    tokens, k = x.shape
    n = base.shape[1]
    adapters, r, _ = a.shape
    if base.shape[0] != tokens or tokens != plan.tokens:
        raise ValueError(f"x {tuple(x.shape)}, base {tuple(base.shape)} and the plan's {plan.tokens} rows do not match")
    if a.shape[2] != k or b.shape != (adapters, n, r) or adapters != plan.adapters:
        raise ValueError(f"a {tuple(a.shape)} / b {tuple(b.shape)} do not match K={k}, N={n}, {plan.adapters} adapters")
    if plan.max_rank > r:
        raise ValueError(f"the plan has rank {plan.max_rank}, the weights hold {r}")
    x_stride, x_last = x.stride()
    base_stride, base_last = base.stride()
    if not a.is_contiguous() or not b.is_contiguous() or x_last != 1 or base_last != 1:
        raise ValueError("a and b must be contiguous, x and base have a contiguous last dimension")
    if scaling is not None and (scaling.dtype != torch.float32 or scaling.shape != (adapters,)
                                or scaling.get_device() != i or not scaling.is_contiguous()):
        raise ValueError(f"scaling must be contiguous float32 [{adapters}] on the plan's device")
    if out is None:
        out, out_stride = torch.empty_strided((tokens, n), (n, 1), dtype=_F16, device=x.device), n
    else:
        if out.dtype != _F16 or out.shape != (tokens, n) or out.get_device() != i or out.stride(1) != 1:
            raise ValueError(f"out must be float16 [{tokens}, {n}] with a contiguous last dimension")
        out_stride = out.stride(0)
    if tokens == 1:                      # a single row's stride says nothing
        x_stride, base_stride, out_stride = k, n, n
    _ADD(_ADD.pack(x.data_ptr(), x_stride, base.data_ptr(), base_stride, out.data_ptr(), out_stride, a.data_ptr(),
                   b.data_ptr(), 0 if scaling is None else scaling.data_ptr(), plan._tiles, plan._rows, plan.n_tiles,
                   plan.tile_rows, tokens, k, n, adapters, r, plan.max_rank, *plan._workspace), plan._current())
    return out

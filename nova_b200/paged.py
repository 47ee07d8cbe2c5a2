"""Paged int8 KV cache for batches of independent requests.

Every request has a length, pages and an open page of its own; a step brings
any number of new tokens for each (one while decoding, a chunk of a prompt,
none).  The storage of a layer is three tensors:

* ``codes``  uint8 ``[num_pages, H_kv, 2, 64, 128]`` (K, V): a page is one
  64-token group of the int8t64 format (``nova_b200.kvquant``), the same codes
  and scales that ``quantize_int8(..., 64, "token")`` gives for finite values
  (one that is not leaves no finite value in its channel of the page);
* ``scales`` fp16 ``[num_pages, H_kv, 4, 128]``: K min, K step, V min, V step;
* ``tails``  fp16 ``[num_tails, H_kv, 2, 64, 128]``: the tokens of pages that
  are not full yet (position p at slot p % 64).

A step of the batch is described once, on the host, by a :class:`PagePlan`;
every layer then runs

    q = qkv_append(qkv, codes, scales, tails, plan, ...)    # norm, RoPE, quantized append
    o = paged_attention(q, codes, scales, tails, plan)      # causal, optional window

:class:`PagedKVCache` owns the tensors of all layers and hands out the pages.
The reference has no counterpart: its caches share one length over the batch
(src/nova/kvattn.py:488-660).  Limits: head_dim 128, 64-token pages, fp16.
"""

from __future__ import annotations

import itertools
from ctypes import addressof, byref
from typing import Sequence

import numpy as np
import torch

from . import _lib

PAGE = 64
HEAD_DIM = 128


def _i64(values, name: str) -> np.ndarray:
    a = np.ascontiguousarray(values, dtype=np.int64)
    if a.ndim != 1:
        raise ValueError(f"{name} must be a flat list of numbers")
    return a


class PagePlan:
    """One step of a batch of requests: where each one's new tokens go and what
    they attend to.

    - ``q_lens``: new tokens of each request (0 allowed); token rows follow one
      another in this order.  ``kv_lens``: cached tokens with them.
    - ``pages``: page numbers of each request, at least ``kv_len // 64``.
    - ``tail_in`` / ``tail_out``: tail buffers of the open page before and after
      the step (any number where there is none).  They are the same while the
      page stays open and differ when another page opens; the next step's
      ``tail_in`` is this one's ``tail_out``.
    - ``windows``: the attention windows that the layers use (0: all keys).
    - ``read_from``: first position that :func:`paged_read` returns, per request
      (default: the start of the first page that the new tokens touch).

    The plan holds device buffers (its work lists, the attention workspace) and
    is used by one stream at a time.  Host lengths are checked here; nothing is
    read back from the device.
    """

    def __init__(self, q_lens: Sequence[int], kv_lens: Sequence[int], pages: Sequence[Sequence[int]], *,
                 tail_in: Sequence[int], tail_out: Sequence[int], num_q_heads: int, num_kv_heads: int,
                 windows: Sequence[int] = (0,), read_from: Sequence[int] | None = None,
                 device: torch.device | str = "cuda") -> None:
        q, kv = _i64(q_lens, "q_lens"), _i64(kv_lens, "kv_lens")
        n = len(q)
        if n == 0 or len(kv) != n or len(pages) != n:
            raise ValueError(f"q_lens, kv_lens and pages must name the same requests ({n}, {len(kv)}, {len(pages)})")
        windows = tuple(int(w) for w in windows)
        if len(windows) > _lib.PAGED_MAX_WINDOWS or len(set(windows)) != len(windows):
            raise ValueError(f"windows must be at most {_lib.PAGED_MAX_WINDOWS} different numbers, got {windows}")
        tin, tout = _i64(tail_in, "tail_in"), _i64(tail_out, "tail_out")
        if len(tin) != n or len(tout) != n:
            raise ValueError("tail_in and tail_out need one buffer per request")
        frm = None if read_from is None else _i64(read_from, "read_from")
        if frm is not None and len(frm) != n:
            raise ValueError("read_from needs one position per request")
        off = np.zeros(n + 1, dtype=np.int64)
        np.cumsum([len(p) for p in pages], out=off[1:])
        flat = np.fromiter(itertools.chain.from_iterable(pages), dtype=np.int64, count=int(off[-1]))

        self.device = torch.device(device)
        self.windows = windows
        a = _lib.PagedPlanArgs()
        a.seqs, a.q_heads, a.kv_heads = n, int(num_q_heads), int(num_kv_heads)
        a.sms = (torch.cuda.get_device_properties(self.device).multi_processor_count
                 if self.device.type == "cuda" else 148)
        a.q_lens, a.kv_lens, a.page_off, a.pages = q.ctypes.data, kv.ctypes.data, off.ctypes.data, flat.ctypes.data
        a.tail_in, a.tail_out = tin.ctypes.data, tout.ctypes.data
        a.read_from = None if frm is None else frm.ctypes.data
        a.n_windows = len(windows)
        a.windows[:len(windows)] = windows
        self.info = _lib.PagedPlanInfo()
        buf = np.empty(4096 + 64 * n + 4 * len(flat), dtype=np.int32)
        _lib.call("nova_paged_plan", byref(a), buf.ctypes.data, buf.size, byref(self.info))
        if self.info.ints > buf.size:
            buf = np.empty(int(self.info.ints), dtype=np.int32)
            _lib.call("nova_paged_plan", byref(a), buf.ctypes.data, buf.size, byref(self.info))
        self.tokens, self.read_rows = int(self.info.tokens), int(self.info.read_rows)
        self.num_q_heads, self.num_kv_heads = int(num_q_heads), int(num_kv_heads)
        self.q_lens, self.kv_lens = q.tolist(), kv.tolist()
        self.tail_out = tout.tolist()
        self.host = buf[:int(self.info.ints)]
        self.buffer = torch.from_numpy(self.host).to(self.device)
        self.workspace = torch.zeros(int(self.info.workspace_bytes), dtype=torch.uint8, device=self.device)
        self._handle = 0                      # on the host: for inspection only
        if self.buffer.is_cuda:               # what csrc/binding.cpp reads (PageHandle)
            self._fields = (_lib.ctypes.c_int64 * 6)(
                addressof(self.info), self.buffer.data_ptr(), self.workspace.data_ptr(), self.workspace.numel(),
                self.buffer.get_device(), _lib.stream_of(self.buffer.device))
            self._handle = _lib.handle(self._fields, _lib.PAGE_PLAN)

    def _on_other_stream(self) -> None:
        """A stream other than the plan's own uses its buffers: the allocator must know."""
        current = torch.cuda.current_stream(self.buffer.device)
        self.buffer.record_stream(current)
        self.workspace.record_stream(current)

    def check_errors(self) -> None:
        """Raises RuntimeError when a bounded wait of an attention launch with
        this plan gave up (its output is then not valid).  Waits for the work of
        every stream of the device: the word is copied by the legacy default
        stream, which does not wait for PyTorch's other streams."""
        torch.cuda.synchronize(self.buffer.device)
        v = _lib.ctypes.c_int(0)
        with torch.cuda.device(self.buffer.device):
            _lib.call("nova_paged_attention_read_error", self.workspace.data_ptr(), byref(v))
        if v.value:
            raise RuntimeError(f"paged attention: a bounded wait gave up (code {v.value})")


def qkv_append(qkv: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, tails: torch.Tensor, plan: PagePlan, *,
               q_norm_weight: torch.Tensor | None = None, k_norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """q|k|v rows of the step's new tokens into the cache, in one launch.

    ``qkv``: fp16 ``[tokens, (H_q + 2 H_kv) * 128]`` (any row stride that is a
    multiple of 8).  Query and key heads get RMSNorm over their 128 channels
    (``q_norm_weight`` / ``k_norm_weight`` fp16 ``[128]``; None: no norm) and
    RoPE at their request's position (``cos`` / ``sin`` fp16 ``[rope_len,
    128]``; None: none), in fp32 and rounded once.  K and V of a page that fills
    are quantized from its 64 tokens, the others stay in ``tails``.  Returns the
    queries, fp16 ``[tokens, H_q, 128]``."""
    return _lib.fast().qkv_append(qkv, codes, scales, tails, plan, q_norm_weight, k_norm_weight, eps, cos, sin, out)


def paged_read(codes: torch.Tensor, scales: torch.Tensor, tails: torch.Tensor, plan: PagePlan
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached K and V of positions ``[read_from, kv_len)`` of every request of
    the plan, as the values they stand for: two fp16 ``[rows, H_kv, 128]``
    tensors, requests one after another."""
    return _lib.fast().paged_read(codes, scales, tails, plan)


def paged_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, tails: torch.Tensor, plan: PagePlan, *,
                    window: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                    lse_out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the step's new tokens over the cache that holds them.

    ``q``: fp16 ``[tokens, H_q, 128]`` (strides that are multiples of 8, last
    dimension contiguous).  The query at position p of a request sees its keys
    ``j <= p`` (``window`` > 0, one of the plan's: also ``j > p - window``).
    ``scale``: of the scores (default ``128 ** -0.5``).  ``lse_out``: fp32
    ``[tokens, H_q]``, log-sum-exp of the scaled scores.  ``out`` may be ``q``.
    Returns fp16 ``[tokens, H_q, 128]``.

    Scores and sums are fp32; weights are fp16 in the second product (with their
    low parts for requests of up to 4 query rows per KV head), so an output is
    within 2^-11 of the sum of its weighted values.  Cached values have to be
    finite: an infinity or NaN in V reaches every query whose work takes in its
    64-token block, with a weight of zero too."""
    return _lib.fast().paged_attention(q, codes, scales, tails, plan, window, scale, out, lse_out)


class PagedKVCache:
    """The paged int8 cache of all layers, and the host side that hands out its
    pages.

        cache = PagedKVCache(num_layers=36, num_kv_heads=8, num_q_heads=32, num_pages=4096, max_requests=64)
        a, b = cache.add(), cache.add()
        plan = cache.plan([a, b], [300, 1])          # a brings 300 tokens, b one
        for layer in range(36):
            q = cache.append(layer, qkv, plan, ...)
            o = cache.attend(layer, q, plan)
        cache.release(a)

    :meth:`plan` reserves the pages and advances the lengths, so every plan it
    returns is to be run once, in order; :meth:`take_back` undoes one that did
    not run to its end.
    """

    def __init__(self, num_layers: int, num_kv_heads: int, num_q_heads: int, num_pages: int, max_requests: int, *,
                 windows: Sequence[int] = (0,), device: torch.device | str = "cuda") -> None:
        if num_q_heads % num_kv_heads:
            raise ValueError(f"q heads {num_q_heads} not divisible by KV heads {num_kv_heads}")
        if min(num_layers, num_kv_heads, num_pages, max_requests) < 1:
            raise ValueError("num_layers, num_kv_heads, num_pages and max_requests must be positive")
        self.num_kv_heads, self.num_q_heads, self.windows = int(num_kv_heads), int(num_q_heads), tuple(windows)
        self.device = torch.device(device)
        shape = (int(num_layers), int(num_pages), self.num_kv_heads)
        self.codes = torch.zeros(*shape, 2, PAGE, HEAD_DIM, dtype=torch.uint8, device=self.device)
        self.scales = torch.zeros(*shape, 4, HEAD_DIM, dtype=torch.float16, device=self.device)
        self.tails = torch.zeros(int(num_layers), 2 * int(max_requests), self.num_kv_heads, 2, PAGE, HEAD_DIM,
                                 dtype=torch.float16, device=self.device)
        self._free = list(range(int(num_pages) - 1, -1, -1))
        self._slots = list(range(int(max_requests) - 1, -1, -1))
        self._requests: dict[int, dict] = {}
        self._next = 0

    def add(self) -> int:
        """A new, empty request; its number."""
        if not self._slots:
            raise RuntimeError("every request slot is in use")
        self._next += 1
        self._requests[self._next] = {"slot": self._slots.pop(), "flip": 0, "length": 0, "pages": []}
        return self._next

    def release(self, request: int) -> None:
        r = self._requests.pop(request)
        self._free.extend(reversed(r["pages"]))
        self._slots.append(r["slot"])

    def length(self, request: int) -> int:
        return self._requests[request]["length"]

    def free_pages(self) -> int:
        return len(self._free)

    def plan(self, requests: Sequence[int], new_tokens: Sequence[int], *, read_from: Sequence[int] | None = None
             ) -> PagePlan:
        """The next step of ``requests``, with ``new_tokens`` for each."""
        if len(set(requests)) != len(requests) or len(new_tokens) != len(requests):
            raise ValueError("plan() takes different requests and one number of new tokens for each")
        rs = [self._requests[i] for i in requests]
        if any(n < 0 for n in new_tokens):
            raise ValueError("new_tokens must not be negative")
        need = [(r["length"] + n) // PAGE - len(r["pages"]) for r, n in zip(rs, new_tokens)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the step needs {sum(need)} pages, {len(self._free)} are free")
        pages = [r["pages"] + self._free[len(self._free) - sum(need[:i + 1]):len(self._free) - sum(need[:i])]
                 for i, r in enumerate(rs)]
        kv = [r["length"] + n for r, n in zip(rs, new_tokens)]
        flips = [r["flip"] ^ (k // PAGE != r["length"] // PAGE) for r, k in zip(rs, kv)]
        plan = PagePlan(list(new_tokens), kv, pages, num_q_heads=self.num_q_heads, num_kv_heads=self.num_kv_heads,
                        tail_in=[2 * r["slot"] + r["flip"] for r in rs],
                        tail_out=[2 * r["slot"] + f for r, f in zip(rs, flips)], windows=self.windows,
                        read_from=read_from, device=self.device)
        del self._free[len(self._free) - sum(need):]
        plan._before = [(i, r, dict(r), p) for i, r, p in zip(requests, rs, pages)]      # what take_back() restores
        for r, k, p, f in zip(rs, kv, pages, flips):
            r["length"], r["pages"], r["flip"] = k, p, f
        return plan

    def take_back(self, plan: PagePlan) -> None:
        """Undoes :meth:`plan` for a step that did not run to its end: its requests
        have the lengths and pages of before, and the step can be planned and run
        again, whatever of it has run (a step leaves the tokens of before as they
        were).  Only for the latest plan of its requests."""
        before = getattr(plan, "_before", None)
        if before is None:
            raise ValueError("not a plan of this cache, or taken back already")
        if any(self._requests.get(i) is not r or r["pages"] is not pages for i, r, _, pages in before):
            raise ValueError("a request of the plan has been planned again or released")
        for _, r, was, pages in reversed(before):
            self._free.extend(pages[len(was["pages"]):])
            r.update(was)
        plan._before = None

    def append(self, layer: int, qkv: torch.Tensor, plan: PagePlan, **kwargs) -> torch.Tensor:
        """:func:`qkv_append` on one layer."""
        return qkv_append(qkv, self.codes[layer], self.scales[layer], self.tails[layer], plan, **kwargs)

    def attend(self, layer: int, q: torch.Tensor, plan: PagePlan, **kwargs) -> torch.Tensor:
        """:func:`paged_attention` on one layer."""
        return paged_attention(q, self.codes[layer], self.scales[layer], self.tails[layer], plan, **kwargs)

    def read(self, layer: int, plan: PagePlan) -> tuple[torch.Tensor, torch.Tensor]:
        """:func:`paged_read` on one layer."""
        return paged_read(self.codes[layer], self.scales[layer], self.tails[layer], plan)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.tails))

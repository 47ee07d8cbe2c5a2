"""A decoder that serves independent requests in one batch.

``NovaDecoder`` advances a batch whose rows share their lengths; here every
request has a prompt, a length, an adapter and output controls of its own, joins
and leaves at any step, and a step may mix prompt chunks with single tokens:

    srv = RequestServer(weights, num_pages=4096, max_requests=64, adapters=bank)
    a = srv.submit(prompt_a, adapter=2, repetition=1.1)
    b = srv.submit(prompt_b, bias={42: -5.0}, allowed=mask_words)
    while ...:
        for request, token in srv.step().items(): ...
    srv.release(a)

One step: embedding rows -> per layer RMSNorm, q|k|v (NF4 GEMM) + adapters
(``lora_add``), norm + RoPE + quantized append (``PagedKVCache.append``), paged
attention, o_proj + adapters, MLP -> lm_head on the rows that finish a prompt or
decode -> ``adjust_logits`` -> ``sample_topk`` -> the token into the request's
history.  The reference's loop serves one request (src/chat.py).
"""

from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field
from itertools import islice
from typing import Mapping, Sequence

import torch

from . import _lib
from .decoder import DecoderConfig, DecoderWeights, NF4Weight, rope_tables
from .kernels import build_nf4_lut, fused_rms_norm, gemm_workspace, nf4_gemm, residual_rms_norm
from .logits import LogitBias, add_generated, add_prompt, adjust_logits, new_history
from .lora import LoraPlan, lora_add
from .paged import PAGE, PagedKVCache, PagePlan
from .quant import nf4_codebook
from .sampling import sample_topk


@dataclass
class AdapterBank:
    """Low-rank adapters of q|k|v and o_proj: ``a`` fp16 ``[adapters, R, K]`` and
    ``b`` fp16 ``[adapters, N, R]`` per layer, ranks on the host, ``scaling`` fp32
    ``[adapters]``."""

    qkv_a: list[torch.Tensor]
    qkv_b: list[torch.Tensor]
    o_a: list[torch.Tensor]
    o_b: list[torch.Tensor]
    ranks: list[int]
    scaling: torch.Tensor

    @classmethod
    def random_init(cls, cfg: DecoderConfig, ranks: Sequence[int], seed: int = 0, device="cuda", std: float = 0.02
                    ) -> "AdapterBank":
        g = torch.Generator(device=device).manual_seed(seed)
        n, r = len(ranks), -(-max(ranks) // 8) * 8

        def pair(out_f, in_f):
            a = (torch.randn(n, r, in_f, generator=g, device=device) * in_f ** -0.5).half()
            return a, (torch.randn(n, out_f, r, generator=g, device=device) * std).half()

        qkv = [pair(cfg.q_dim + 2 * cfg.kv_dim, cfg.hidden_size) for _ in range(cfg.num_hidden_layers)]
        o = [pair(cfg.hidden_size, cfg.q_dim) for _ in range(cfg.num_hidden_layers)]
        return cls([p[0] for p in qkv], [p[1] for p in qkv], [p[0] for p in o], [p[1] for p in o], list(ranks),
                   torch.ones(n, dtype=torch.float32, device=device))


@dataclass
class _Request:
    cache_id: int
    slot: int
    adapter: int
    todo: deque = field(default_factory=deque)   # prompt tokens that are not in the cache yet


class RequestError(RuntimeError):
    """A step that cannot be taken because of some of its requests: ``requests``
    are those to change, to release or to leave out of ``step(requests)``."""

    def __init__(self, message: str, requests: Sequence[int]) -> None:
        super().__init__(message.format(list(requests)))
        self.requests = list(requests)


class RequestServer:
    """Serves requests over a paged cache.  ``chunk``: the most prompt tokens that
    a request brings into one step.  Sampling settings are the batch's;
    ``temperature`` 0 is greedy."""

    def __init__(self, weights: DecoderWeights, num_pages: int, max_requests: int, *, adapters: AdapterBank | None = None,
                 chunk: int = 512, max_len: int = 32768, temperature: float = 0.0, top_k: int = 64, top_p: float = 1.0,
                 seed: int = 0, device="cuda") -> None:
        cfg = weights.cfg
        if chunk < 1 or max_requests < 1:
            raise ValueError("chunk and max_requests must be positive")
        self.w, self.cfg, self.adapters, self.chunk, self.max_len = weights, cfg, adapters, int(chunk), int(max_len)
        self.device = torch.device(device)
        self.temperature, self.top_k, self.top_p = temperature, top_k, top_p
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.cache = PagedKVCache(cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.num_attention_heads, num_pages,
                                  max_requests, device=device)
        self.lut = build_nf4_lut(weights.code if weights.code is not None else nf4_codebook()).to(self.device)
        self.cos, self.sin = rope_tables(self.max_len, cfg.head_dim, cfg.rope_theta, self.device)
        shapes = [(cfg.q_dim + 2 * cfg.kv_dim, cfg.hidden_size), (cfg.hidden_size, cfg.q_dim),
                  (2 * cfg.intermediate_size, cfg.hidden_size), (cfg.hidden_size, cfg.intermediate_size),
                  (cfg.vocab_size, cfg.hidden_size)]
        self.gemm_ws = max((gemm_workspace(self.device, n, k) for n, k in shapes), key=lambda t: t.numel()).clone()
        # controls and state of every slot
        n, v = int(max_requests), cfg.vocab_size
        self.history = new_history(n, v, self.device)
        self.repetition = torch.ones(n, dtype=torch.float32, device=self.device)
        self.frequency = torch.zeros(n, dtype=torch.float32, device=self.device)
        self.presence = torch.zeros(n, dtype=torch.float32, device=self.device)
        self.masks = torch.full((n, -(-v // 32)), -1, dtype=torch.int32, device=self.device)
        self.tokens = torch.zeros(n, dtype=torch.int64, device=self.device)     # last token of each slot
        self.biases: list[dict] = [{} for _ in range(n)]
        self.masked: list[bool] = [False] * n
        self._free = list(range(n - 1, -1, -1))
        self._requests: dict[int, _Request] = {}
        self.logits: torch.Tensor | None = None      # of the last step, after the controls
        self.raw_logits: torch.Tensor | None = None

    def submit(self, prompt: Sequence[int], *, adapter: int = -1, repetition: float = 1.0, frequency: float = 0.0,
               presence: float = 0.0, bias: Mapping[int, float] | None = None, allowed: torch.Tensor | None = None) -> int:
        """A new request; its number.  ``allowed``: int32 bit mask ``[ceil(vocab /
        32)]`` of the tokens that may follow (:meth:`set_allowed` changes it)."""
        prompt, adapter = [int(t) for t in prompt], int(adapter)
        repetition, frequency, presence = float(repetition), float(frequency), float(presence)
        bias = {int(t): float(v) for t, v in (bias or {}).items()}
        if not prompt or min(prompt) < 0 or max(prompt) >= self.cfg.vocab_size:
            raise ValueError("the prompt must hold at least one token, all within the vocabulary")
        if len(prompt) > self.max_len:
            raise ValueError(f"a prompt of {len(prompt)} tokens is longer than max_len {self.max_len}")
        if adapter >= (len(self.adapters.ranks) if self.adapters else 0):
            raise ValueError(f"no adapter {adapter}")
        if not repetition > 0:
            raise ValueError("repetition must be positive")
        if bias and (min(bias) < 0 or max(bias) >= self.cfg.vocab_size):
            raise ValueError("bias tokens must lie within the vocabulary")
        if allowed is not None:
            self._check_mask(allowed)
        rid = self.cache.add()
        slot = self._free.pop()
        self._requests[rid] = _Request(rid, slot, adapter, deque(prompt))
        self.history[slot].zero_()
        ids = torch.tensor(prompt, dtype=torch.int64, device=self.device)
        add_prompt(self.history[slot:slot + 1], ids, torch.tensor([0, len(prompt)], dtype=torch.int32, device=self.device))
        self.repetition[slot], self.frequency[slot], self.presence[slot] = repetition, frequency, presence
        self.biases[slot] = bias
        self.masked[slot] = allowed is not None
        if allowed is not None:
            self.masks[slot].copy_(allowed)
        return rid

    def _check_mask(self, allowed: torch.Tensor) -> None:
        if not torch.is_tensor(allowed) or allowed.dtype != torch.int32 or allowed.shape != self.masks.shape[1:]:
            raise ValueError(f"allowed must be int32 [{self.masks.shape[1]}]")

    def set_allowed(self, request: int, allowed: torch.Tensor | None) -> None:
        """The tokens that may follow from now on (a grammar's next state); None: all."""
        slot = self._requests[request].slot
        if allowed is not None:
            self._check_mask(allowed)
            self.masks[slot].copy_(allowed)
        self.masked[slot] = allowed is not None

    def release(self, request: int) -> None:
        r = self._requests.pop(request)
        self.cache.release(r.cache_id)
        self._free.append(r.slot)

    def length(self, request: int) -> int:
        """Cached tokens of a request."""
        return self.cache.length(request)

    def _linear(self, x: torch.Tensor, w: NF4Weight, epilogue: int = _lib.NF4_PLAIN, residual: torch.Tensor | None = None,
                half: bool = False) -> torch.Tensor:
        out = torch.empty(x.shape[0], w.n // 2 if half else w.n, dtype=torch.float16, device=self.device)
        return nf4_gemm(x, w.tc_units(), self.lut, out, n=w.n, epilogue=epilogue, residual=residual, workspace=self.gemm_ws)

    def step(self, requests: Sequence[int] | None = None) -> dict[int, int]:
        """One forward pass of ``requests`` (default: all): the next chunk of each
        unfinished prompt, the last token of every other.  Returns the new token
        of each request whose prompt is complete.  A step that raises leaves every
        request as it was before (draws of the sampler excepted).  It raises
        :class:`RequestError` for requests that would pass ``max_len``, that need
        more pages than are free, or whose mask and biases leave no token, and
        RuntimeError where a kernel reports that its result is not valid."""
        rids = list(self._requests) if requests is None else list(requests)
        if not rids:
            return {}
        rs = [self._requests[i] for i in rids]
        counts = [min(len(r.todo), self.chunk) or 1 for r in rs]
        have = [self.cache.length(i) for i in rids]
        past = [i for i, h, n in zip(rids, have, counts) if h + n > self.max_len]
        if past:
            raise RequestError(f"requests {{}} would pass max_len {self.max_len}", past)
        need = {i: (h + n) // PAGE - h // PAGE for i, h, n in zip(rids, have, counts)}
        if sum(need.values()) > self.cache.free_pages():
            raise RequestError(f"requests {{}} need {sum(need.values())} pages, {self.cache.free_pages()} are free",
                               [i for i in rids if need[i]])
        plan = self.cache.plan(rids, counts)
        try:
            done, tok, mine, history, report = self._forward(rs, counts, plan)
            report = report.tolist()                         # the step has run
            words, tokens, ruled_out = report[:2], report[2:2 + len(done)], report[2 + len(done):]
            if any(words):
                self._raise_errors(plan)
            if any(ruled_out):
                raise RequestError("no token is left for requests {}: their masks and biases rule out all",
                                   [rids[i] for i, out in zip(done, ruled_out) if out])
        except BaseException:
            self.cache.take_back(plan)
            raise
        for r, n in zip(rs, counts):
            for _ in range(n if r.todo else 0):
                r.todo.popleft()
        if done:
            self.history[mine] = history
            self.tokens[mine] = tok
        return {rids[i]: t for i, t in zip(done, tokens)}

    def _raise_errors(self, plan: PagePlan) -> None:
        """Raises RuntimeError, and clears the error words, where a bounded wait of the step's attention or GEMM
        kernels gave up: its tokens, and what it put into the cache, are not valid then."""
        code = _lib.ctypes.c_int(0)
        with torch.cuda.device(self.device):                 # the server's workspace first: it outlives the plan's
            _lib.call("nova_nf4_gemm_read_error", self.gemm_ws.data_ptr(), _lib.ctypes.byref(code))
        plan.check_errors()
        if code.value:
            raise RuntimeError(f"NF4 GEMM: a bounded wait gave up (code {code.value})")

    def _forward(self, rs: list[_Request], counts: list[int], plan: PagePlan) -> tuple:
        """The step's kernels: which of ``rs`` get a token, those tokens, their slots, their histories with the tokens,
        and one tensor for the host: the error words of attention and GEMM, the tokens, and whether each one is ruled
        out (logit -inf, so every other is too).  Of the server's state only the cache's memory changes."""
        fresh = [list(islice(r.todo, n)) if r.todo else None for r, n in zip(rs, counts)]
        cfg, bank = self.cfg, self.adapters
        slots = torch.tensor([r.slot for r in rs], dtype=torch.int64, device=self.device)
        ids = torch.tensor([t for f in fresh for t in (f or [0])], dtype=torch.int64, device=self.device)
        decoding = [i for i, f in enumerate(fresh) if f is None]
        starts = [sum(counts[:i]) for i in range(len(counts))]
        if decoding:
            at = torch.tensor([starts[i] for i in decoding], dtype=torch.int64, device=self.device)
            ids[at] = self.tokens[slots[torch.tensor(decoding, device=self.device)]]
        lora = LoraPlan(counts, [r.adapter for r in rs], bank.ranks, device=self.device) if bank else None

        x = self.w.embed[ids]
        for li, w in enumerate(self.w.layers):
            xn = fused_rms_norm(x, w.input_ln, cfg.rms_norm_eps)
            qkv = self._linear(xn, w.qkv)
            if bank:
                lora_add(xn, qkv, bank.qkv_a[li], bank.qkv_b[li], lora, scaling=bank.scaling, out=qkv)
            q = self.cache.append(li, qkv, plan, q_norm_weight=w.q_norm, k_norm_weight=w.k_norm, eps=cfg.rms_norm_eps,
                                  cos=self.cos, sin=self.sin)
            o = self.cache.attend(li, q, plan).view(-1, cfg.q_dim)
            y = self._linear(o, w.o)
            if bank:
                lora_add(o, y, bank.o_a[li], bank.o_b[li], lora, scaling=bank.scaling, out=y)
            x, xn = residual_rms_norm(y, x, w.post_ln, cfg.rms_norm_eps)
            act = self._linear(xn, w.gate_up, _lib.NF4_SILU_MUL, half=True)
            x = self._linear(act, w.down, _lib.NF4_RESIDUAL, residual=x)

        words = (plan.workspace[:4].view(torch.int32), self.gemm_ws[4:8].view(torch.int32))
        done = [i for i, r in enumerate(rs) if len(r.todo) <= counts[i]]
        if not done:
            return [], None, None, None, torch.cat(words)
        last = torch.tensor([starts[i] + counts[i] - 1 for i in done], dtype=torch.int64, device=self.device)
        mine = slots[torch.tensor(done, dtype=torch.int64, device=self.device)]
        self.raw_logits = self._linear(fused_rms_norm(x[last], self.w.final_norm, cfg.rms_norm_eps), self.w.lm_head)
        which = [rs[i].slot for i in done]
        entries = [self.biases[s] for s in which]
        allowed_row = torch.tensor([s if self.masked[s] else -1 for s in which], dtype=torch.int32, device=self.device)
        history = self.history[mine]
        self.logits = adjust_logits(
            self.raw_logits, history=history, repetition=self.repetition[mine], frequency=self.frequency[mine],
            presence=self.presence[mine], bias=LogitBias(entries, cfg.vocab_size, self.device) if any(entries) else None,
            allowed=self.masks, allowed_row=allowed_row)
        u = torch.rand(len(done), generator=self.gen, device=self.device) if self.temperature > 0 else None
        tok = sample_topk(self.logits, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, uniform=u)
        ruled_out = self.logits.gather(1, tok[:, None])[:, 0] == -float("inf")
        report = torch.cat((*words, tok, ruled_out))
        add_generated(history, tok)
        return done, tok, mine, history, report

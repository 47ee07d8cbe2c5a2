"""Measured cases of the operators that serve a batch of independent requests.

A decode step of one model shape (Qwen3-VL-4B: 32 query heads on 8 KV heads of
128 channels, hidden size 2560, vocabulary 151936) over requests that each have
a length, pages, an adapter and output controls of their own:

* ``append``: q|k|v rows of ragged new tokens -> per-head RMSNorm + RoPE, K and
  V into a paged cache that is quantized to int8 as each 64-token page fills
  (asymmetric, per channel over the page; the open page stays fp16), and the
  touched pages read back;
* ``attention``: the new tokens (one per request, or a chunk) over that cache;
* ``lora``: the low-rank adapters of the requests, added to a shared
  projection's output;
* ``logits``: repetition / frequency / presence penalties, token biases and
  grammar masks.

``run`` computes them in elementary torch operations in fp32 (``own`` false) or
through ``nova_b200`` (``own`` true) on the same tensors.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
D = 128            # head_dim
PAGE = 64          # tokens per page
EPS = 1e-6


# --------------------------------------------------------------------- cases

def listed():
    att = {"op": "attention", "kv_heads": 8, "group": 4, "window": 0}
    app = {"op": "append", "kv_heads": 8, "group": 4}
    return [
        # the first tokens after a short prompt, one user: latency alone
        {"name": "attn_decode_1x77", **att, "decode": 1, "chunks": 0, "q": 1, "ctx_lo": 77, "ctx": 77, "salt": 0},
        # an ordinary serving batch: 16 conversations of very different lengths
        {"name": "attn_decode_16x8192", **att, "decode": 16, "chunks": 0, "q": 1, "ctx_lo": 40, "ctx": 8191,
         "salt": 1},
        # a large batch of long documents: the cache is far larger than L2
        {"name": "attn_decode_32x32768", **att, "decode": 32, "chunks": 0, "q": 1, "ctx_lo": 8000, "ctx": 32768,
         "salt": 2},
        # the next 509 tokens of a prompt over 8192 cached ones
        {"name": "attn_chunk_509_8192", **att, "decode": 0, "chunks": 1, "q": 509, "ctx_lo": 8192, "ctx": 8192,
         "salt": 3},
        # prompt chunks of several requests in one batch with decoding ones
        {"name": "attn_mixed_6x600_10x5000", **att, "decode": 10, "chunks": 6, "q": 601, "ctx_lo": 3, "ctx": 5000,
         "salt": 4},
        # a large chunk at the end of a long document
        {"name": "attn_chunk_2048_30011", **att, "decode": 0, "chunks": 1, "q": 2048, "ctx_lo": 30011, "ctx": 30011,
         "salt": 5},
        # one token of each of 64 requests enters the cache
        {"name": "append_decode_64", **app, "seqs": 64, "q_lo": 1, "q": 1, "ctx_lo": 30, "ctx": 8000, "salt": 6},
        # ragged prompt chunks of 8 requests enter the cache
        {"name": "append_chunk_8x1021", **app, "seqs": 8, "q_lo": 130, "q": 1021, "ctx_lo": 1, "ctx": 4000,
         "salt": 7},
        # 64 decoding requests with 24 adapters of rank up to 16 beside the q|k|v projection
        {"name": "lora_decode_64_r16", "op": "lora", "seqs": 64, "q_lo": 1, "q": 1, "adapters": 24, "rank": 16,
         "k": 2560, "n": 6144, "salt": 8},
        # prompt chunks of 5 requests with adapters of rank up to 64 beside the gate|up projection
        {"name": "lora_chunk_5x700_r64", "op": "lora", "seqs": 5, "q_lo": 90, "q": 701, "adapters": 4, "rank": 64,
         "k": 2560, "n": 19456, "salt": 9},
        # one request's next-token logits
        {"name": "logits_1", "op": "logits", "rows": 1, "vocab": 151936, "bias": 20, "masks": 1, "salt": 10},
        # the logits of 64 requests, half of them under a grammar
        {"name": "logits_64", "op": "logits", "rows": 64, "vocab": 151936, "bias": 300, "masks": 8, "salt": 11},
    ]


def _log(rng, lo, hi):
    v = int(round(lo * (hi / lo) ** rng.random()))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "lora", "logits"])
    salt = rng.randrange(1000)
    if op == "attention":
        kind = rng.choice(["decode", "chunk", "mixed"])
        hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        c = {"op": op, "kv_heads": hkv, "group": group, "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
             "decode": 0, "chunks": 0, "q": 1, "salt": salt}
        ctx = _log(rng, 1, 32768)
        if kind in ("decode", "mixed"):
            c["decode"] = _log(rng, 1, 48)
        if kind in ("chunk", "mixed"):
            c["chunks"], c["q"] = _log(rng, 1, 6), _log(rng, 2, 2048)
        c["ctx"], c["ctx_lo"] = ctx, _log(rng, 1, ctx)
        # no more than the largest listed cases: scores of the padded batch, and cached bytes
        n = c["decode"] + c["chunks"]
        while n * hkv * group * c["q"] * (c["ctx"] + c["q"]) > 1.2e9 or n * hkv * (c["ctx"] + c["q"]) > 4.0e6:
            c["ctx"], c["q"] = max(1, c["ctx"] * 3 // 4), max(1 + (c["chunks"] > 0), c["q"] * 3 // 4)
            c["ctx_lo"] = min(c["ctx_lo"], c["ctx"])
        return c
    if op == "append":
        q = rng.choice([1, 1, _log(rng, 2, 1500)])
        return {"op": op, "kv_heads": rng.choice([1, 2, 4, 8]), "group": rng.choice([1, 2, 3, 4, 8]),
                "seqs": _log(rng, 1, 64 if q == 1 else 8), "q": q, "q_lo": _log(rng, 1, q), "ctx_lo": 1,
                "ctx": _log(rng, 1, 8000), "salt": salt}
    if op == "lora":
        q = rng.choice([1, 1, _log(rng, 2, 700)])
        return {"op": op, "seqs": _log(rng, 1, 64 if q == 1 else 5), "q": q, "q_lo": _log(rng, 1, q),
                "adapters": _log(rng, 1, 24), "rank": rng.choice([8, 16, 32, 64]),
                "k": rng.choice([2560, 4096, 9728]), "n": rng.choice([1024, 2560, 4096, 6144, 19456]), "salt": salt}
    return {"op": op, "rows": _log(rng, 1, 64), "vocab": rng.choice([151936, 32000, 50257, _log(rng, 1000, 150000)]),
            "bias": rng.choice([0, _log(rng, 1, 300)]), "masks": rng.choice([0, 1, 4, 8]), "salt": salt}


def _spread(n, lo, hi, salt):
    """n whole numbers over [lo, hi], even over the logarithm; the first is hi."""
    lo = min(lo, hi)
    return [hi if i == 0 else int(round(lo * (hi / lo) ** ((0.6180339887 * i + 0.37 * salt) % 1.0))) for i in range(n)]


def _lengths(case):
    """(new tokens, length after them) of each request of an attention or append case."""
    if case["op"] == "append":
        q = _spread(case["seqs"], case["q_lo"], case["q"], case["salt"])
        past = _spread(case["seqs"], case["ctx_lo"], case["ctx"], case["salt"] + 1)
        return q, [a + b for a, b in zip(q, past)]
    q = _spread(case["chunks"], 2, case["q"], case["salt"]) if case["chunks"] else []
    past = _spread(case["chunks"], case["ctx_lo"], case["ctx"], case["salt"] + 1) if case["chunks"] else []
    kv = [a + b for a, b in zip(q, past)]
    if case["decode"]:
        q += [1] * case["decode"]
        kv += _spread(case["decode"], case["ctx_lo"], case["ctx"], case["salt"] + 2)
    return q, kv


def _adapters(case):
    """(tokens, adapter or -1 for none) of each request, and the adapters' ranks."""
    n, salt = case["adapters"], case["salt"]
    tokens = _spread(case["seqs"], case["q_lo"], case["q"], salt)
    which = [-1 if (i + salt) % 8 == 5 else (i * 7 + salt) % n for i in range(case["seqs"])]
    ranks = [case["rank"] if i % 3 == 0 else max(1, case["rank"] // 2 + (i * 5 + salt) % (case["rank"] // 2 + 1))
             for i in range(n)]
    return tokens, which, ranks


def _seen_pairs(q, kv, window):
    """(query, key) pairs of one request under the causal mask and the window."""
    first = kv - q
    if not window:
        return q * first + q * (q + 1) // 2
    full = max(0, min(q, kv - max(first, window)))      # queries that see a whole window
    rest = q - full
    return full * window + rest * first + rest * (rest + 1) // 2


def work(case):
    op = case["op"]
    if op in ("attention", "append"):
        hkv, hq = case["kv_heads"], case["kv_heads"] * case["group"]
        q, kv = _lengths(case)
    if op == "attention":
        w = case["window"]
        seen = [min(n, w + m - 1) if w else n for m, n in zip(q, kv)]       # keys that some query reads
        full = [min(s, n // PAGE * PAGE - (n - s)) if n // PAGE * PAGE > n - s else 0 for s, n in zip(seen, kv)]
        cache = sum(f * 2 * D + (s - f) * 4 * D + math.ceil(f / PAGE) * 4 * D * 2 for f, s in zip(full, seen)) * hkv
        pairs = sum(_seen_pairs(m, n, w) for m, n in zip(q, kv))
        return {"bytes": cache + 2 * sum(q) * hq * D * 2, "flops": 4 * D * hq * pairs}
    if op == "append":
        t = sum(q)
        rows = t * (hq + 2 * hkv) * D * 2 + t * hq * D * 2 + 2 * t * D * 2       # q|k|v in, q out, cos and sin
        old = touched = full = 0
        for m, n in zip(q, kv):
            first = (n - m) // PAGE * PAGE
            touched += n - first
            if n // PAGE * PAGE > first:
                full += n // PAGE * PAGE - first
                old += n - m - first                     # open-page tokens that a page takes over
        opened = touched - full
        page = full * 2 * D + full // PAGE * 4 * D * 2
        tail = min(t, opened) * 4 * D
        return {"bytes": rows + hkv * (old * 4 * D + page + tail                 # written
                                       + page + opened * 4 * D + touched * 4 * D),   # read back
                "flops": t * (hq + hkv) * D * 8}
    if op == "lora":
        tokens, which, ranks = _adapters(case)
        used = sum(ranks[a] for a in set(which) if a >= 0)
        t = sum(tokens)
        busy = [(m, ranks[a]) for m, a in zip(tokens, which) if a >= 0]
        return {"bytes": sum(m for m, _ in busy) * case["k"] * 2 + 2 * t * case["n"] * 2
                + used * (case["k"] + case["n"]) * 2,
                "flops": sum(2 * m * r * (case["k"] + case["n"]) for m, r in busy)}
    rows, v = case["rows"], case["vocab"]
    return {"bytes": rows * v * 6 + min(rows, case["masks"]) * v // 8 + rows * case["bias"] * 8, "flops": rows * v * 8}


# ------------------------------------------------------------------- prepare

def _randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).half()


def _int(values):
    return torch.tensor(values, dtype=torch.int64, device=DEV)


def _cache(g, q, kv, hkv, spare=3):
    """A paged cache holding the requests' tokens: scattered pages with codes and
    scales as normed keys and values leave them, and open pages in fp16."""
    full = [n // PAGE for n in kv]
    total = sum(full) + spare
    codes = torch.empty(total, hkv, 2, PAGE, D, dtype=torch.uint8, device=DEV)
    codes.copy_(torch.randint(0, 128, codes.shape, generator=g, device=DEV, dtype=torch.uint8))
    codes += torch.randint(0, 128, codes.shape, generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.empty(total, hkv, 4, D, dtype=torch.float16, device=DEV)
    loud = 1.0 + 7.0 * (torch.rand(1, hkv, 1, D, generator=g, device=DEV) < 0.03)     # a few loud key channels
    step = (0.012 + 0.012 * torch.rand(total, hkv, 2, D, generator=g, device=DEV))
    step[:, :, :1] *= loud
    low = -step * (127.0 + 10.0 * torch.randn(total, hkv, 2, D, generator=g, device=DEV))
    scales[:, :, 0::2], scales[:, :, 1::2] = low.half(), step.half()
    tails = _randn(g, 2 * len(kv), hkv, 2, PAGE, D, scale=0.8)
    order = torch.randperm(total, generator=g, device=DEV).tolist()
    table, at = [], 0
    for f in full:
        table.append(order[at:at + f])
        at += f
    tail_in = [2 * i for i in range(len(kv))]
    tail_out = [2 * i + (n // PAGE != (n - m) // PAGE) for i, (m, n) in enumerate(zip(q, kv))]
    return codes, scales, tails, table, tail_in, tail_out


def _plan(s, case):
    """The plan that the framework's program keeps for a step (all layers use it)."""
    from nova_b200.paged import PagePlan
    s["plan"] = PagePlan(s["q_lens"], s["kv_lens"], s["table"], tail_in=s["tail_in"], tail_out=s["tail_out"],
                         num_q_heads=case["kv_heads"] * case["group"], num_kv_heads=case["kv_heads"],
                         windows=(case.get("window", 0),), device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return {"attention": _prepare_attention, "append": _prepare_append, "lora": _prepare_lora,
            "logits": _prepare_logits}[case["op"]](case, g)


def _prepare_attention(case, g):
    q, kv = _lengths(case)
    hkv, group = case["kv_heads"], case["group"]
    codes, scales, tails, table, tail_in, tail_out = _cache(g, q, kv, hkv)
    s = {"op": "attention", "codes": codes, "scales": scales, "tails": tails, "table": table, "tail_in": tail_in,
         "tail_out": tail_out, "q_lens": q, "kv_lens": kv, "window": case["window"],
         "q": _randn(g, sum(q), hkv * group, D, scale=1.2)}
    if own:
        _plan(s, case)
    else:
        wide, most = max(1, max(len(t) for t in table)), max(q)
        starts = [sum(q[:i]) for i in range(len(q))]
        s["pages"] = _int([t + [0] * (wide - len(t)) for t in table])
        s["buffer"], s["length"], s["news"] = _int(tail_out), _int(kv), _int(q)
        s["row"] = _int([[a + min(j, max(m - 1, 0)) for j in range(most)] for a, m in zip(starts, q)])
    return s


def _prepare_append(case, g):
    q, kv = _lengths(case)
    hkv, hq = case["kv_heads"], case["kv_heads"] * case["group"]
    codes, scales, tails, table, tail_in, tail_out = _cache(g, q, kv, hkv)
    angle = (torch.arange(max(kv), device=DEV).double()[:, None]
             * 5e6 ** (-torch.arange(0, D, 2, device=DEV).double() / D)[None])
    angle = torch.cat([angle, angle], 1)
    s = {"op": "append", "codes": codes, "scales": scales, "tails": tails, "table": table, "tail_in": tail_in,
         "tail_out": tail_out, "q_lens": q, "kv_lens": kv, "kv_heads": hkv,
         "qkv": _randn(g, sum(q), (hq + 2 * hkv) * D, scale=2.0),
         "q_norm": 1.0 + _randn(g, D, scale=0.2), "k_norm": 1.0 + _randn(g, D, scale=0.2),
         "cos": angle.cos().half(), "sin": angle.sin().half()}
    if own:
        _plan(s, case)
    else:
        # which token each place of each touched page comes from
        pos, page, out_buf, old, new, there, slot_at = [], [], [], [], [], [], []
        t0 = 0
        for i, (m, n) in enumerate(zip(q, kv)):
            pos += range(n - m, n)
            for p in range((n - m) // PAGE, -(-n // PAGE)):
                page.append(table[i][p] if (p + 1) * PAGE <= n else -1)
                out_buf.append(tail_out[i])
                at = [p * PAGE + j for j in range(PAGE)]
                old.append([tail_in[i] if x < n - m else -1 for x in at])
                new.append([t0 + x - (n - m) if n - m <= x < n else 0 for x in at])
                there.append([x < n for x in at])
            t0 += m
        s["pos"], s["page"], s["out_buf"] = _int(pos), _int(page), _int(out_buf)
        s["old"], s["new"], s["there"] = _int(old), _int(new), _int(there).bool()
    return s


def _prepare_lora(case, g):
    tokens, which, ranks = _adapters(case)
    n, r, k, width = case["adapters"], case["rank"], case["k"], case["n"]
    t = sum(tokens)
    s = {"op": "lora", "x": _randn(g, t, k), "base": _randn(g, t, width),
         "a": _randn(g, n, r, k, scale=k ** -0.5), "b": _randn(g, n, width, r, scale=r ** -0.5),
         "scaling": 0.5 + torch.rand(n, generator=g, device=DEV)}
    if own:
        from nova_b200.lora import LoraPlan
        s["plan"] = LoraPlan(tokens, which, ranks, device=DEV)
    else:
        s["which"] = _int([a for m, a in zip(tokens, which) for _ in range(m)])
        s["ranks"] = _int(ranks)
    return s


def _prepare_logits(case, g):
    rows, v, masks = case["rows"], case["vocab"], case["masks"]
    logits = _randn(g, rows, v, scale=3.0)
    logits[:, v // 3] = -math.inf                                  # a token that the model itself rules out
    history = (torch.rand(rows, v, generator=g, device=DEV) < 0.004).to(torch.int16)
    history *= torch.randint(1, 9, (rows, v), generator=g, device=DEV).to(torch.int16)
    prompt = torch.rand(rows, v, generator=g, device=DEV) < 0.01
    history += torch.where(prompt, -32768, 0).to(torch.int16)      # top bit: in the prompt; low bits: times generated
    s = {"op": "logits", "logits": logits, "history": history,
         "repetition": 1.0 + 0.3 * torch.rand(rows, generator=g, device=DEV),
         "frequency": 0.5 * torch.rand(rows, generator=g, device=DEV),
         "presence": 0.5 * torch.rand(rows, generator=g, device=DEV),
         "vocab": v, "allowed": None, "allowed_row": None, "bias": None}
    if masks:
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (masks, -(-v // 32)), generator=g, device=DEV).to(torch.int32)
        s["allowed_row"] = torch.tensor([(i * 3) % masks if i % 2 == 0 else -1 for i in range(rows)],
                                        dtype=torch.int32, device=DEV)
        logits[0, ::97] = math.nan                                 # what a masked or allowed token may hold
    entries = []
    if case["bias"]:
        pick = torch.rand(rows, case["bias"], generator=g, device=DEV).tolist()
        size = torch.randn(rows, case["bias"], generator=g, device=DEV).mul(4).tolist()
        entries = [{int(p * v): w for p, w in zip(*row)} if i % 4 != 1 else {} for i, row in enumerate(zip(pick, size))]
    if own:
        if entries:
            from nova_b200.logits import LogitBias
            s["bias"] = LogitBias(entries, v, device=DEV)
    elif entries:
        s["bias"] = (_int([i for i, e in enumerate(entries) for _ in e]), _int([t for e in entries for t in e]),
                     torch.tensor([w for e in entries for w in e.values()], dtype=torch.float32, device=DEV))
    s["entries"] = entries
    return s


# ----------------------------------------------------------------------- run

def run(s):
    if own:
        return _run_own(s)
    return {"attention": _attention, "append": _append, "lora": _lora, "logits": _logits}[s["op"]](s)


def _run_own(s):
    if s["op"] == "attention":
        from nova_b200.paged import paged_attention
        return paged_attention(s["q"], s["codes"], s["scales"], s["tails"], s["plan"], window=s["window"])
    if s["op"] == "append":
        from nova_b200.paged import paged_read, qkv_append
        q = qkv_append(s["qkv"], s["codes"], s["scales"], s["tails"], s["plan"], q_norm_weight=s["q_norm"],
                       k_norm_weight=s["k_norm"], eps=EPS, cos=s["cos"], sin=s["sin"])
        return (q, *paged_read(s["codes"], s["scales"], s["tails"], s["plan"]))
    if s["op"] == "lora":
        from nova_b200.lora import lora_add
        return lora_add(s["x"], s["base"], s["a"], s["b"], s["plan"], scaling=s["scaling"])
    from nova_b200.logits import adjust_logits
    return adjust_logits(s["logits"], history=s["history"], repetition=s["repetition"], frequency=s["frequency"],
                         presence=s["presence"], bias=s["bias"], allowed=s["allowed"], allowed_row=s["allowed_row"])


def _stored(codes, scales, j):
    """The values that codes of K (j = 0) or V (j = 1) stand for, in fp32: fp16(code * step + min)."""
    x = codes[..., j, :, :].float() * scales[..., 2 * j + 1, :].float().unsqueeze(-2)
    return (x + scales[..., 2 * j, :].float().unsqueeze(-2)).half().float()


def _attention(s):
    q, pages = s["q"].float(), s["pages"]
    hkv, hq = s["codes"].shape[1], q.shape[1]
    n, group = len(s["q_lens"]), hq // hkv
    whole = (s["length"] // PAGE * PAGE)[:, None]
    at = torch.arange(pages.shape[1] * PAGE, device=DEV).expand(n, -1)
    open_at = whole + torch.arange(PAGE, device=DEV)
    pos = torch.cat([at.masked_fill(at >= whole, 2 ** 31), open_at.masked_fill(open_at >= s["length"][:, None], 2 ** 31)],
                    1)                                                                    # [n, keys]
    k, v = ((torch.cat([_stored(s["codes"][pages], s["scales"][pages], j).transpose(1, 2).flatten(2, 3),
                        s["tails"][s["buffer"], :, j].float()], 2)) for j in (0, 1))      # [n, hkv, keys, D]
    rows = s["row"].shape[1]
    qp = q[s["row"]].view(n, rows, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * rows, D)
    score = (qp @ k.transpose(2, 3)).view(n, hkv, group, rows, -1) * D ** -0.5
    qpos = (s["length"] - s["news"])[:, None] + torch.arange(rows, device=DEV)            # [n, rows]
    hide = pos[:, None, :] > qpos[:, :, None]
    if s["window"]:
        hide |= pos[:, None, :] <= qpos[:, :, None] - s["window"]
    score.masked_fill_(hide[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = score.exp_()
    p /= p.sum(-1, keepdim=True)
    v = v.masked_fill((pos > 2 ** 30)[:, None, :, None], 0.0)
    o = (p.view(n, hkv, group * rows, -1) @ v).view(n, hkv, group, rows, D).permute(0, 3, 1, 2, 4)
    live = torch.arange(rows, device=DEV) < s["news"][:, None]
    return o.reshape(n, rows, hq, D)[live].half()


def _rope(x, cos, sin):
    turned = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
    return x * cos + turned * sin


def _append(s):
    hkv = s["kv_heads"]
    x = s["qkv"].float().view(s["qkv"].shape[0], -1, D)
    hq = x.shape[1] - 2 * hkv
    cos, sin = s["cos"][s["pos"]].float()[:, None], s["sin"][s["pos"]].float()[:, None]
    qk = x[:, :hq + hkv]
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    q = _rope(qk[:, :hq] * s["q_norm"].float(), cos, sin).half()
    kv = torch.stack([_rope(qk[:, hq:] * s["k_norm"].float(), cos, sin), x[:, hq + hkv:]], 2).half()   # [T, hkv, 2, D]
    # every touched page's tokens: from the open page as it was, or new
    slot = torch.arange(PAGE, device=DEV).expand_as(s["old"])
    was = s["tails"][s["old"].clamp_min(0), :, :, slot]                                # [pages, PAGE, hkv, 2, D]
    got = torch.where((s["old"] >= 0)[..., None, None, None], was, kv[s["new"]])
    closed = s["page"] >= 0
    f = got.float()
    low, high = f.amin(1), f.amax(1)                                                   # [pages, hkv, 2, D]
    step = ((high - low) / 255.0).clamp_min(1e-8)
    code = ((f - low[:, None]) / step[:, None]).round().clamp(0, 255).to(torch.uint8)
    s["codes"][s["page"][closed]] = code[closed].permute(0, 2, 3, 1, 4)
    s["scales"][s["page"][closed]] = torch.stack([low, step], 3).flatten(2, 3)[closed].half()
    live = s["there"] & ~closed[:, None]
    s["tails"][s["out_buf"][:, None].expand_as(slot)[live], :, :, slot[live]] = got[live]
    # the touched pages as the cache now holds them
    page, buf = s["page"].clamp_min(0), s["out_buf"]
    back = []
    for j in (0, 1):
        held = _stored(s["codes"][page], s["scales"][page], j).half()                  # [pages, hkv, PAGE, D]
        x = torch.where(closed[:, None, None, None], held, s["tails"][buf, :, j])
        back.append(x.transpose(1, 2)[s["there"]])
    return (q, *back)


def _lora(s):
    n, r, k = s["a"].shape
    h = s["x"].float() @ s["a"].float().view(n * r, k).t()
    mine = (s["which"][:, None, None] == torch.arange(n, device=DEV)[None, :, None])
    mine = mine & (torch.arange(r, device=DEV)[None, None] < s["ranks"][None, :, None])
    h = (h.view(-1, n, r) * s["scaling"][None, :, None]).masked_fill(~mine, 0.0).view(-1, n * r)
    return (s["base"].float() + h @ s["b"].float().transpose(1, 2).reshape(n * r, -1)).half()


def _logits(s):
    x, h = s["logits"].float(), s["history"].int()
    times = h & 0x7FFF
    rep = s["repetition"][:, None]
    x = torch.where(h != 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * times - s["presence"][:, None] * (times > 0)
    if s["bias"] is not None:
        x.index_put_(s["bias"][:2], s["bias"][2], accumulate=True)
    if s["allowed"] is not None:
        at = torch.arange(s["vocab"], device=DEV)
        bit = (s["allowed"][s["allowed_row"].clamp_min(0).long()][:, at // 32] >> (at % 32)) & 1
        x = x.masked_fill((bit == 0) & (s["allowed_row"] >= 0)[:, None], -math.inf)
    return x.half()


# --------------------------------------------------------------------- exact

def exact(case, seed):
    """What run() returns for these inputs, from the definitions, in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attention": _exact_attention, "append": _exact_append, "lora": _exact_lora,
            "logits": _exact_logits}[case["op"]](s)


def _exact_pages(s, i, head, j, count):
    """Stored fp16 values of the first `count` pages of request i, one head, in 64 bits."""
    ids = _int(s["table"][i][:count])
    c = s["codes"][ids, head, j].double()
    low, step = s["scales"][ids, head, 2 * j].double(), s["scales"][ids, head, 2 * j + 1].double()
    return (c * step[:, None] + low[:, None]).half().double().reshape(-1, D)


def _exact_attention(s):
    hkv, hq = s["codes"].shape[1], s["q"].shape[1]
    g = hq // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    t0 = 0
    for i, (m, n) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        behind = torch.arange(n - m, n, device=DEV)[:, None] - torch.arange(n, device=DEV)[None]
        hide = behind < 0
        if s["window"]:
            hide |= behind >= s["window"]
        for h in range(hkv):
            k, v = (torch.cat([_exact_pages(s, i, h, j, n // PAGE),
                               s["tails"][s["tail_out"][i], h, j, :n % PAGE].double()]) for j in (0, 1))
            for e in range(h * g, (h + 1) * g):
                a = (s["q"][t0:t0 + m, e].double() @ k.t()) / math.sqrt(D)
                out[t0:t0 + m, e] = torch.softmax(a.masked_fill(hide, -math.inf), 1) @ v
        t0 += m
    return out


def _exact_append(s):
    hkv = s["kv_heads"]
    x = s["qkv"].double().view(s["qkv"].shape[0], -1, D)
    hq = x.shape[1] - 2 * hkv
    new = [None, None]
    roped = []
    for part, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hkv], s["k_norm"])):
        y = part / (part.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        c, z = s["cos"][s["pos"]].double()[:, None], s["sin"][s["pos"]].double()[:, None]
        first, second = y[..., :D // 2], y[..., D // 2:]
        roped.append(torch.cat([first * c[..., :D // 2] - second * z[..., :D // 2],
                                second * c[..., D // 2:] + first * z[..., D // 2:]], -1))
    new = (roped[1].half().double(), x[:, hq + hkv:])
    read = ([], [])
    t0 = 0
    for i, (m, n) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        past = (n - m) % PAGE
        for j in (0, 1):
            old = s["tails"][s["tail_in"][i], :, j, :past].double().transpose(0, 1)
            tok = torch.cat([old, new[j][t0:t0 + m]])                                  # from the first touched page on
            whole = tok.shape[0] // PAGE * PAGE
            p = tok[:whole].view(-1, PAGE, hkv, D)
            low, high = (p.amin(1, keepdim=True), p.amax(1, keepdim=True)) if whole else (p[:, :1], p[:, :1])
            step = ((high - low) / 255).clamp_min(1e-8)
            code = ((p - low) / step).round().clamp(0, 255)
            held = (code * step.half().double() + low.half().double()).half().double().view(whole, hkv, D)
            read[j].append(torch.cat([held, tok[whole:]]))
        t0 += m
    return (roped[0], torch.cat(read[0]), torch.cat(read[1]))


def _exact_lora(s):
    out = s["base"].double()
    for a, rank in enumerate(s["ranks"].tolist()):
        mine = s["which"] == a
        h = s["x"][mine].double() @ s["a"][a, :rank].double().t()
        out[mine] += float(s["scaling"][a]) * (h @ s["b"][a, :, :rank].double().t())
    return out


def _exact_logits(s):
    out = []
    for i in range(s["logits"].shape[0]):
        x, h = s["logits"][i].double(), s["history"][i].long()
        rep = s["repetition"][i].double()
        times = torch.where(h < 0, h + 32768, h)
        x = torch.where(h == 0, x, torch.where(x > 0, x / rep, x * rep))
        x = x - s["frequency"][i].double() * times - s["presence"][i].double() * (times != 0)
        for_row = s["entries"][i] if s["entries"] else {}
        if for_row:
            x[_int(list(for_row))] += torch.tensor(list(for_row.values()), dtype=torch.float32, device=DEV).double()
        if s["allowed"] is not None and int(s["allowed_row"][i]) >= 0:
            words = s["allowed"][int(s["allowed_row"][i])].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32, device=DEV)) & 1
            x = torch.where(bits.flatten()[:s["vocab"]] == 1, x, torch.full_like(x, -math.inf))
        out.append(x)
    return torch.stack(out)

"""Plain 64-bit forms of the paged-cache operators for the tests, and the error
bounds that the kernels' arithmetic has against them."""

from __future__ import annotations

import torch

PAGE, D = 64, 128


class State:
    """A paged cache of one layer holding random tokens for ragged requests,
    with pages scattered over the pool."""

    def __init__(self, q_lens, kv_lens, kv_heads, q_heads, seed=0, spare=2, scale=0.8):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.hkv, self.hq = list(q_lens), list(kv_lens), kv_heads, q_heads
        full = [n // PAGE for n in kv_lens]
        total = sum(full) + spare
        self.codes = torch.randint(0, 256, (total, kv_heads, 2, PAGE, D), generator=g, dtype=torch.uint8)
        step = (0.004 + 0.012 * torch.rand(total, kv_heads, 2, D, generator=g)) * scale
        low = -step * (127.0 + 20.0 * torch.randn(total, kv_heads, 2, D, generator=g))
        self.scales = torch.stack([low[:, :, 0], step[:, :, 0], low[:, :, 1], step[:, :, 1]], 2).half()
        self.tails = (torch.randn(2 * len(full), kv_heads, 2, PAGE, D, generator=g) * scale).half()
        order = torch.randperm(total, generator=g).tolist()
        self.pages, at = [], 0
        for f in full:
            self.pages.append(order[at:at + f])
            at += f
        self.tail_in = [2 * i for i in range(len(full))]
        self.tail_out = [2 * i + (n // PAGE != (n - m) // PAGE) for i, (m, n) in enumerate(zip(q_lens, kv_lens))]
        self.q = torch.randn(sum(q_lens), q_heads, D, generator=g).half()
        self.gen = g

    def plan(self, **kw):
        from nova_b200.paged import PagePlan

        kw.setdefault("num_q_heads", self.hq)
        return PagePlan(self.q_lens, self.kv_lens, self.pages, tail_in=self.tail_in, tail_out=self.tail_out,
                        num_kv_heads=self.hkv, **kw)

    def values(self, i, head, j):
        """Stored K (j = 0) or V (j = 1) of request i, one head: [kv_len, D] in 64 bits."""
        n = self.kv_lens[i]
        ids = self.pages[i][:n // PAGE]
        c = self.codes[ids, head, j].double()
        low, step = self.scales[ids, head, 2 * j].double(), self.scales[ids, head, 2 * j + 1].double()
        x = (c * step[:, None] + low[:, None]).half().double().reshape(-1, D)
        return torch.cat([x, self.tails[self.tail_out[i], head, j, :n % PAGE].double()])


def attention(s: State, window=0, scale=D ** -0.5, device="cpu"):
    """(out, bound on the kernel's error, lse, bound on its error), 64 bits.

    The kernel rounds each weight to fp16 (2^-11 of it at most; a weight below
    the normal range is off by at most 2^-25 of the largest one, which is 1 or
    more) and the result once more; scores are fp32 sums of 128 exact products
    (at most 128 * 2^-24 of the sum of their magnitudes) and exp2 and the sums
    over keys add a few 2^-22.  A score error e moves a weight and the sum of
    weights by a factor of e each."""
    out, bound = torch.zeros(s.q.shape, dtype=torch.float64), torch.zeros(s.q.shape, dtype=torch.float64)
    lse = torch.full(s.q.shape[:2], -float("inf"), dtype=torch.float64)
    lse_bound = torch.zeros(s.q.shape[:2], dtype=torch.float64)
    t0, gq = 0, s.hq // s.hkv
    out, bound, lse, lse_bound = (t.to(device) for t in (out, bound, lse, lse_bound))
    for i, (m, n) in enumerate(zip(s.q_lens, s.kv_lens)):
        if not m:
            continue
        behind = torch.arange(n - m, n, device=device)[:, None] - torch.arange(n, device=device)[None]
        hide = (behind < 0) | ((behind >= window) if window else torch.zeros_like(behind, dtype=torch.bool))
        for h in range(s.hkv):
            k, v = s.values(i, h, 0).to(device), s.values(i, h, 1).to(device)
            for e in range(h * gq, (h + 1) * gq):
                q = s.q[t0:t0 + m, e].to(device).double()
                a = (q @ k.t() * scale).masked_fill(hide, -float("inf"))
                size = (q.abs() @ k.abs().t() * scale).masked_fill(hide, 0.0).amax(1, keepdim=True)
                p = torch.softmax(a, 1)
                o, mass = p @ v, p @ v.abs()
                err = 2 * (128 * 2.0 ** -24 * size + 2.0 ** -22 * (4 + a.abs().masked_fill(hide, 0.0).amax(1, keepdim=True)))
                out[t0:t0 + m, e] = o
                under = 2.0 ** -25 * (~hide).sum(1, keepdim=True) * v.abs().max() * p.amax(1, keepdim=True)
                bound[t0:t0 + m, e] = 2.0 ** -11 * o.abs() + 2.0 ** -24 + (2.0 ** -11 + err + n * 2.0 ** -24) * mass + under
                lse[t0:t0 + m, e] = torch.logsumexp(a, 1)
                lse_bound[t0:t0 + m, e] = (err + n * 2.0 ** -24)[:, 0] + 2.0 ** -22 * (1 + lse[t0:t0 + m, e].abs())
        t0 += m
    return out.cpu(), bound.cpu(), lse.cpu(), lse_bound.cpu()


def norm_rope(x, w, cos, sin, eps):
    """(rows after RMSNorm and RoPE, magnitude of the terms), 64 bits: x [T, heads, D], cos / sin [T, D]."""
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is None:
        return y, y.abs()
    c, z = cos.double()[:, None], sin.double()[:, None]
    turned = torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1)
    return y * c + turned * z, (y * c).abs() + (turned * z).abs()

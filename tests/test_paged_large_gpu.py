"""GPU: paged attention at the sizes where the work is cut -- several segments
per CTA, tiles cut between CTAs, many splits, both kernels in one call -- and
page offsets past 2^31 bytes, against 64 bits (bounds in paged_reference.py)."""

from __future__ import annotations

import random

import pytest
import torch

import paged_reference as ref
from test_paged_gpu import close, run_attention

pytestmark = pytest.mark.gpu

PAGE, D = 64, 128


@pytest.mark.parametrize("q_lens,kv_lens,hkv,hq,window", [
    ([2000], [9000], 2, 8, 0),                      # tiles cut between CTAs
    ([300, 1000, 64, 1, 1, 33], [4000, 1000, 6000, 8000, 100, 33], 8, 32, 0),   # many segments per CTA, both kernels
    ([700, 650, 1], [5000, 700, 3000], 4, 20, 1000),
    ([129, 257, 513], [129, 300, 5000], 1, 1, 0),   # one head: 128-row halves end inside a tile
    ([1] * 40, [50 + 97 * i for i in range(40)], 2, 16, 0),
    ([2, 1, 8, 1, 3], [30000, 20000, 10000, 64, 3], 2, 8, 0),                   # up to 32 splits
    ([9, 10, 11], [700, 1500, 90], 2, 6, 0),        # 27 to 33 rows: either side of the kernels' boundary
    ([40], [2500], 3, 24, 64),
])
def test_attention(cuda_lib, q_lens, kv_lens, hkv, hq, window):
    s = ref.State(q_lens, kv_lens, hkv, hq, seed=sum(kv_lens))
    out, lse = run_attention(s, window)
    want, bound, want_lse, lse_bound = ref.attention(s, window, device="cuda")
    close(out, want, bound, "out")
    close(lse, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(cuda_lib, seed):
    rng = random.Random(seed)
    hkv = rng.choice([1, 2, 3, 4])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    n = rng.randint(1, 12)
    q = [rng.choice([0, 1, 1, 1, rng.randint(2, 40), rng.randint(2, 600)]) for _ in range(n)]
    kv = [m + rng.choice([0, rng.randint(0, 64), rng.randint(0, 4000)]) for m in q]
    if not sum(q):
        q[0], kv[0] = 1, max(kv[0], 1)
    window = rng.choice([0, 0, rng.randint(1, 300)])
    s = ref.State(q, kv, hkv, hq, seed=seed)
    out, lse = run_attention(s, window)
    want, bound, want_lse, lse_bound = ref.attention(s, window, device="cuda")
    close(out, want, bound, f"{q} {kv} {hkv} {hq} {window}")
    close(lse, want_lse, lse_bound, "lse")


def test_growing_maximum(cuda_lib):
    """Scores that keep growing along the keys, by far more than the rescaling threshold each step, and keys
    that dwarf all others at either end."""
    s = ref.State([300], [1500], 1, 4, seed=1, scale=0.2)
    g = torch.Generator().manual_seed(3)
    direction = torch.randn(D, generator=g)
    direction /= direction.norm()
    full = 1500 // PAGE
    ramp = torch.linspace(0.0, 40.0, full)
    for p in range(full):
        low = s.scales[s.pages[0][p], 0, 0].float() + ramp[p] * direction
        s.scales[s.pages[0][p], 0, 0] = low.half()
    s.scales[s.pages[0][0], 0, 0] += (60.0 * direction).half()
    s.q = (s.q.float() * 0.2 + 8.0 * direction).half()
    out, lse = run_attention(s)
    want, bound, want_lse, lse_bound = ref.attention(s)
    close(out, want, bound, "out")
    close(lse, want_lse, lse_bound, "lse")


def test_page_offsets_past_2_31_bytes(cuda_lib):
    """Pages at the end of a 2.2 GB pool: append, read back and attend with both kernels."""
    from nova_b200.paged import PagePlan, paged_attention, paged_read, qkv_append

    hkv, hq, pages = 8, 16, 17000
    s = ref.State([1, 100], [300, 1000], hkv, hq, seed=2)
    shift = pages - s.codes.shape[0]
    codes = torch.zeros(pages, hkv, 2, PAGE, D, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(pages, hkv, 4, D, dtype=torch.float16, device="cuda")
    codes[shift:], scales[shift:] = s.codes.cuda(), s.scales.cuda()
    tails = s.tails.cuda()
    plan = PagePlan(s.q_lens, s.kv_lens, [[p + shift for p in x] for x in s.pages], tail_in=s.tail_in, tail_out=s.tail_out,
                    num_q_heads=hq, num_kv_heads=hkv, read_from=[0, 0])
    want, bound, _, _ = ref.attention(s)
    close(paged_attention(s.q.cuda(), codes, scales, tails, plan), want, bound, "out")
    k, v = paged_read(codes, scales, tails, plan)
    for j, x in enumerate((k, v)):
        assert torch.equal(x[:300].cpu().double(), torch.stack([s.values(0, h, j) for h in range(hkv)], 1))
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(101, (hq + 2 * hkv) * D, generator=g).half()
    q = qkv_append(qkv.cuda(), codes, scales, tails, plan)
    assert torch.equal(q.cpu(), qkv.view(101, -1, D)[:, :hq])
    assert not codes[:shift].any()
    k, v = paged_read(codes, scales, tails, plan)
    new = qkv.view(101, -1, D)[1:, hq + hkv:]
    open_tokens = 1000 % PAGE
    assert torch.equal(v[-open_tokens:].cpu(), new[-open_tokens:])
    step = scales[plan_pages(plan, 1)[-1], :, 3].float().cpu()
    closed = new[:100 - open_tokens][-PAGE:].float()
    got = v[300 + 1000 - open_tokens - PAGE:300 + 1000 - open_tokens].float().cpu()
    assert ((got[-closed.shape[0]:] - closed).abs() <= 0.51 * step + 2.0 ** -9 * closed.abs() + 2.0 ** -10).all()


def plan_pages(plan, i):
    seq = plan.host[plan.info.seq_off + 8 * i:plan.info.seq_off + 8 * i + 8]
    return plan.host[plan.info.page_off + seq[3]:plan.info.page_off + seq[3] + seq[2] // PAGE].tolist()

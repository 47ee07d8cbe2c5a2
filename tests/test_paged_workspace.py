"""The attention workspace of a plan: one set of arrival counters that no
schedule's partials reach, whatever windows the layers take in turn."""

from __future__ import annotations

import random

import pytest
import torch

import paged_reference as ref
from nova_b200.paged import PAGE, PagePlan
from test_paged_gpu import close
from test_paged_plan import make

PART_FLOATS, TILE_PART_FLOATS = 132, 256 * 130        # of a few-rows partial's row, of a cut tile's partial


def layout(plan):
    """([counter ranges], [ranges of partials]) in bytes over all schedules of a plan."""
    counters, parts = [], []
    heads = plan.num_kv_heads
    for s in plan.info.sched[:plan.info.n_windows]:
        for r in s.rows:
            counters.append((r.counters_off, r.counters_off + r.n_parts * heads * 4))
            parts.append((r.parts_off, r.parts_off + r.n_parts * heads * r.rows_per_tile * PART_FLOATS * 4))
        parts.append((s.tile_parts_off, s.tile_parts_off + s.n_tile_parts * TILE_PART_FLOATS * 4))
    return counters, parts


def check_layout(plan):
    counters, parts = layout(plan)
    head, total = plan.info.head_bytes, plan.info.workspace_bytes
    assert 256 <= head <= total and head % 256 == 0
    for a, b in counters:
        assert 256 <= a <= b <= head                   # past the error word, within the zeroed head
    for a, b in parts:
        assert head <= a <= b <= total and a % 256 == 0
    for s in range(plan.info.n_windows):               # within a schedule nothing overlaps
        mine = sorted(r for r in counters[2 * s:2 * s + 2] + parts[3 * s:3 * s + 3] if r[0] < r[1])
        assert all(x[1] <= y[0] for x, y in zip(mine, mine[1:]))
    return counters, parts


@pytest.mark.parametrize("q,kv,hq,hkv,windows", [
    ([1] * 8, [32768] * 8, 32, 8, (0, 1024)),
    ([300, 1, 1], [4000, 3000, 2000], 32, 8, (0, 128)),
    ([1, 64], [600, 400], 8, 2, (0, 128, 37)),
    ([512, 1], [4000, 3000], 32, 8, (0, 1024, 64, 1)),
    ([1], [1], 1, 1, (0,)),
    ([0, 0], [64, 0], 4, 1, ()),
])
def test_partials_never_reach_the_counters(q, kv, hq, hkv, windows):
    counters, _ = check_layout(make(q, kv, hq, hkv, windows=windows))
    if len(windows) > 1:
        assert max(b - a for a, b in counters) > 0     # some schedule does count arrivals


def test_partials_never_reach_the_counters_at_random():
    rng = random.Random(3)
    for _ in range(200):
        hkv = rng.choice([1, 2, 4, 8])
        q = [rng.choice([0, 1, 1, 2, rng.randint(1, 700)]) for _ in range(rng.randint(1, 9))]
        kv = [m + rng.choice([0, rng.randint(0, 20000)]) for m in q]
        windows = tuple(rng.sample([0, 1, 37, 128, 1024, 5000], rng.randint(1, 4)))
        check_layout(make(q, kv, hkv * rng.choice([1, 3, 4, 8]), hkv, windows=windows))


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens,hkv,hq", [
    ([1, 64], [600, 400], 2, 8),
    ([1] * 6, [8000, 3000, 5000, 700, 64, 1], 2, 8),          # splits of single tokens
    ([2, 1, 8], [6000, 4000, 5000], 2, 8),                    # both few-rows lists
    ([400, 1, 90], [5000, 6000, 2500], 2, 8),                 # cut tiles and splits
])
def test_layers_take_their_windows_in_turn(cuda_lib, q_lens, kv_lens, hkv, hq):
    """One plan and its one workspace over layers whose windows alternate, each result whole and right."""
    from nova_b200.paged import paged_attention

    windows = (0, 128, 37)
    s = ref.State(q_lens, kv_lens, hkv, hq, seed=17)
    plan = s.plan(windows=windows)
    check_layout(plan)
    cache, q = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda()), s.q.cuda()
    want = {w: ref.attention(s, w, device="cuda") for w in windows}
    first = {}
    for w in (0, 128, 0, 37, 0, 128, 37, 37, 128, 0):
        out = torch.full_like(q, float("nan"))
        lse = torch.full(q.shape[:2], float("nan"), dtype=torch.float32, device="cuda")
        paged_attention(q, *cache, plan, window=w, out=out, lse_out=lse)
        close(out, *want[w][:2], f"out of window {w}")
        close(lse, *want[w][2:], f"lse of window {w}")
        assert torch.equal(out, first.setdefault(w, out)), f"window {w} repeats bit for bit"
    plan.check_errors()
    assert not plan.workspace[:plan.info.head_bytes].any()    # ready for the next launch


@pytest.mark.gpu
def test_cache_serves_alternating_layers(cuda_lib):
    """PagedKVCache(windows=(0, w)): full and windowed layers over one plan per step, with decoding steps."""
    from nova_b200.paged import PagedKVCache

    hkv, hq, layers, w = 2, 8, 4, 100
    cache = PagedKVCache(layers, hkv, hq, num_pages=64, max_requests=2, windows=(0, w))
    a, b = cache.add(), cache.add()
    g = torch.Generator(device="cuda").manual_seed(9)
    kv = [0, 0]
    for m in ([1500, 70], [1, 1], [1, 130], [1, 1]):
        plan = cache.plan([a, b], m)
        kv = [x + y for x, y in zip(kv, m)]
        x = torch.randn(sum(m), (hq + 2 * hkv) * 128, generator=g, device="cuda").half()
        for layer in range(layers):
            q = cache.append(layer, x, plan)
            got = cache.attend(layer, q, plan, window=w if layer % 2 else 0)
            alone = PagePlan(m, kv, [cache._requests[r]["pages"] for r in (a, b)],
                             tail_in=plan.tail_out, tail_out=plan.tail_out, num_q_heads=hq, num_kv_heads=hkv,
                             windows=(w if layer % 2 else 0,)) if same_page(m, kv) else None
            if alone is not None:                             # a fresh plan and workspace: the same bits
                assert torch.equal(got, cache.attend(layer, q, alone, window=w if layer % 2 else 0))
            assert torch.isfinite(got).all()
        plan.check_errors()


def same_page(m, kv):
    return all((n - k) // PAGE == n // PAGE for k, n in zip(m, kv))

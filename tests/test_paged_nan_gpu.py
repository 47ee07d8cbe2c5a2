"""GPU: paged attention of queries that are not finite: their rows say so, output
and log-sum-exp, and no other row changes."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_lens,kv_lens,hkv,hq", [
    ([1], [40], 1, 4),               # a single work item
    ([1, 2], [3000, 200], 2, 8),     # splits
    ([150], [150], 2, 8),            # whole tiles
    ([70], [5000], 2, 8),            # cut tiles, joined
])
def test_rows_that_are_not_finite(cuda_lib, q_lens, kv_lens, hkv, hq):
    from nova_b200.paged import paged_attention

    s = ref.State(q_lens, kv_lens, hkv, hq, seed=21)
    plan, cache = s.plan(), (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())

    def run(q):
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
        return paged_attention(q, *cache, plan, lse_out=lse), lse

    q = s.q.cuda()
    clean = run(q)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    q[0, 1, 5], bad[0, 1] = float("nan"), True
    q[-1, -1, 100], bad[-1, -1] = float("inf"), True
    out, lse = run(q)
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(out[~bad], clean[0][~bad]) and torch.equal(lse[~bad], clean[1][~bad])
    plan.check_errors()

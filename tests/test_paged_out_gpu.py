"""GPU: where paged attention writes: every layout whose rows are apart, q itself,
and no layout whose rows overlap."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

D = 128


def setup(q_lens, kv_lens, hkv=2, hq=8):
    s = ref.State(q_lens, kv_lens, hkv, hq, seed=31)
    return s.q.cuda(), (s.codes.cuda(), s.scales.cuda(), s.tails.cuda()), s.plan()


def test_rows_that_overlap_are_refused(cuda_lib):
    from nova_b200.paged import paged_attention

    q, cache, plan = setup([1, 2], [70, 130])
    buf = torch.empty(3 * 8 * D, dtype=torch.float16, device="cuda")
    for out in (buf[:8 * D].view(1, 8, D).expand(3, 8, D), buf[:3 * D].view(3, 1, D).expand(3, 8, D),
                buf.as_strided((3, 8, D), (8, D, 1)), buf.as_strided((3, 8, D), (8 * D, 64, 1)),
                buf.as_strided((3, 8, D), (D, D, 1)), buf.as_strided((3, 8, D), (7 * D, D, 1)),
                buf.as_strided((3, 8, D), (D, 2 * D, 1))):
        with pytest.raises(ValueError, match="overlap"):
            paged_attention(q, *cache, plan, out=out)


def test_layouts_that_are_apart(cuda_lib):
    from nova_b200.paged import paged_attention

    for q_lens, kv_lens, hkv, hq in (([1, 2], [70, 130], 2, 8), ([1], [70], 1, 4), ([1, 1], [9, 70], 1, 1), ([1], [9], 1, 1),
                                     ([90], [500], 2, 8)):
        q, cache, plan = setup(q_lens, kv_lens, hkv, hq)
        t = q.shape[0]
        want = paged_attention(q, *cache, plan)
        rows = torch.empty(t, hq + 1, 2 * D, dtype=torch.float16, device="cuda")
        heads = torch.empty(hq, t + 1, D + 8, dtype=torch.float16, device="cuda")
        for out in (rows[:, 1:, :D], heads[:, :t, 8:].transpose(0, 1)):
            assert torch.equal(paged_attention(q, *cache, plan, out=out), want)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 3], [5000, 200]), ([200, 1], [3000, 700])])
def test_out_may_be_q(cuda_lib, q_lens, kv_lens):
    """A row is written once all who read it have: by the CTA that joins its splits, by the join kernel, or by the
    only CTA that has it."""
    from nova_b200.paged import paged_attention

    q, cache, plan = setup(q_lens, kv_lens)
    want = paged_attention(q, *cache, plan)
    for _ in range(5):
        mine = q.clone()
        assert paged_attention(mine, *cache, plan, out=mine).data_ptr() == mine.data_ptr() and torch.equal(mine, want)

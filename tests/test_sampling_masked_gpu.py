"""GPU: sampling from rows of which a mask has left few tokens, at draws next to
one, where the running sum of the probabilities can round to less than the draw."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("left", [1, 2, 3, 7, 40])
def test_a_masked_token_is_never_drawn(cuda_lib, left):
    from nova_b200.sampling import sample_topk

    rows, v = 4000, 512
    g = torch.Generator().manual_seed(left)
    logits = torch.full((rows, v), -float("inf"), dtype=torch.float16)
    allowed = torch.stack([torch.randperm(v, generator=g)[:left] for _ in range(rows)])
    logits.scatter_(1, allowed, torch.randn(rows, left, generator=g).half() * 3)
    for u in (0.0, 0.5, 1 - 2.0 ** -22, 1 - 2.0 ** -24):
        tok = sample_topk(logits.cuda(), temperature=0.9, top_k=64, top_p=1.0,
                          uniform=torch.full((rows,), u, device="cuda")).cpu()
        assert (allowed == tok[:, None]).any(1).all(), f"{(~(allowed == tok[:, None]).any(1)).sum()} forbidden tokens at {u}"

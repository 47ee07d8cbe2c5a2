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


def test_infinite_logits(cuda_lib):
    """A logit of +inf (a bias beyond fp16's range) is taken with certainty, several of them alike."""
    from nova_b200.logits import LogitBias, adjust_logits
    from nova_b200.sampling import sample_topk

    rows, v = 64, 1000
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(rows, v, generator=g).half()
    forced = torch.randint(0, v, (rows,), generator=g)
    biased = adjust_logits(logits.cuda(), bias=LogitBias([{int(t): 1e6} for t in forced], v))
    u = torch.rand(rows, generator=g).cuda()
    for temperature in (0.0, 0.7, 2.0):
        tok = sample_topk(biased, temperature=temperature, top_k=50, top_p=0.9, uniform=u)
        assert torch.equal(tok.cpu(), forced)
    two = logits.clone()
    two[:, 10] = two[:, 20] = float("inf")
    tok = sample_topk(two.cuda(), temperature=1.0, top_k=50, top_p=1.0, uniform=torch.linspace(0, 0.999, rows).cuda()).cpu()
    assert torch.equal(tok, torch.where(torch.linspace(0, 0.999, rows) < 0.5, 10, 20))

"""GPU: the repetition penalty divides and multiplies as its formula does, bit for
bit in fp32, at any size of the penalty."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rep", [1.0, 1.1, 1.3, 3.0, 7.7, 0.3, 1e-39, 3e38])
def test_repetition_is_a_division(cuda_lib, rep):
    from nova_b200.logits import adjust_logits

    rows, v = 3, 5003
    g = torch.Generator().manual_seed(2)
    x = torch.randn(rows, v, generator=g) * 5
    x[0, :50] = torch.randn(50, generator=g) * 1e-38            # subnormal numbers among them
    hist = (torch.rand(rows, v, generator=g) < 0.5).to(torch.int16)
    r = torch.full((rows,), rep)
    want = torch.where(hist != 0, torch.where(x > 0, x / r[:, None], x * r[:, None]), x)
    got = adjust_logits(x.cuda(), history=hist.cuda(), repetition=r.cuda()).cpu()
    assert torch.equal(got, want)

"""GPU: the serving operators on a device that is not the current one."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref
from test_paged_gpu import close

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[0, 1])
def device(request, cuda_lib):
    """Every device of up to two, the other one being current."""
    if torch.cuda.device_count() <= request.param:
        pytest.skip("one GPU")
    with torch.cuda.device((request.param + 1) % torch.cuda.device_count()):
        yield torch.device("cuda", request.param)


def test_paged_operators(device):
    from nova_b200.paged import paged_attention, paged_read, qkv_append

    s = ref.State([1, 90, 3], [3000, 150, 70], 2, 8, seed=9)
    want, bound, _, _ = ref.attention(s)
    plan = s.plan(device=device)
    cache = [t.to(device) for t in (s.codes, s.scales, s.tails)]
    current = torch.cuda.current_device()
    out = paged_attention(s.q.to(device), *cache, plan)
    assert out.device == device and torch.cuda.current_device() == current
    close(out, want, bound, "out")
    q = qkv_append(torch.randn(94, 12 * 128, device=device).half(), *cache, plan)
    k, v = paged_read(*cache, plan)
    plan.check_errors()
    assert q.device == k.device == v.device == device and torch.cuda.current_device() == current


def test_lora_and_logits(device):
    from nova_b200.logits import LogitBias, add_generated, adjust_logits, new_history
    from nova_b200.lora import LoraPlan, lora_add

    x, base = torch.ones(3, 64, device=device).half(), torch.zeros(3, 32, device=device).half()
    a, b = torch.ones(1, 8, 64, device=device).half(), torch.ones(1, 32, 8, device=device).half()
    out = lora_add(x, base, a, b, LoraPlan([3], [0], [8], device=device))
    assert (out == 512).all()
    h = new_history(2, 100, device)
    add_generated(h, torch.tensor([5, 7], device=device))
    assert int(h[0, 5]) == int(h[1, 7]) == 1 and int(h.sum()) == 2
    got = adjust_logits(torch.zeros(2, 100, device=device), history=h, presence=torch.ones(2, device=device),
                        bias=LogitBias([{9: 2.0}, {}], 100, device))
    want = torch.zeros(2, 100)
    want[0, 5] = want[1, 7] = -1
    want[0, 9] = 2
    assert torch.equal(got.cpu(), want)

"""GPU: values that are not finite in a page that fills.  By the format's
definition (minimum and maximum over the page's 64 tokens, per channel) such a
channel of the page holds no finite value; nothing else changes."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

D = 128


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("token", [0, 70, 127, 130])      # of 140: in the first two pages, in the open one
def test_no_finite_value_stands_for_one_that_is_not(cuda_lib, bad, token):
    from nova_b200.paged import paged_read, qkv_append

    hkv, hq, n = 2, 4, 140
    s = ref.State([n], [n], hkv, hq, seed=5)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(n, (hq + 2 * hkv) * D, generator=g).half().cuda()

    def run(x):
        cache = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())
        plan = s.plan(read_from=[0])
        qkv_append(x, *cache, plan)
        return paged_read(*cache, plan)

    k, v = run(x)
    y = x.clone()
    y[token, (hq + 1) * D + 3] = bad                      # K, head 1, channel 3
    y[token, (hq + hkv) * D + 100] = bad                  # V, head 0, channel 100
    for clean, got, head, channel in ((k, run(y)[0], 1, 3), (v, run(y)[1], 0, 100)):
        hit = torch.zeros_like(clean, dtype=torch.bool)
        page = slice(token // 64 * 64, token // 64 * 64 + 64) if token < 128 else slice(token, token + 1)
        hit[page, head, channel] = True
        assert not torch.isfinite(got[hit]).any()
        assert torch.equal(got[~hit], clean[~hit])

"""GPU: the serving operators on streams other than the one that made their
plans and lists."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

LONG = 60_000_000      # clock cycles of a kernel that only waits: about 30 ms


def test_check_errors_waits_for_other_streams(cuda_lib):
    """An error word that a launch on another stream sets late is seen, and cleared once it has been."""
    plan = ref.State([1], [70], 1, 1).plan()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    word = plan.workspace[:4].view(torch.int32)
    for late in (1, LONG):                                    # first with all kernels loaded: loading may wait itself
        with torch.cuda.stream(side):
            torch.cuda._sleep(late)
            word.fill_(7)                                     # what a bounded wait that gives up leaves
        with pytest.raises(RuntimeError, match="code 7"):
            plan.check_errors()
        plan.check_errors()


def others_memory(ptr, nbytes, count=64):
    """Whether any of `count` fresh allocations of that size on the current stream lies in [ptr, ptr + nbytes)."""
    fresh = [torch.empty(nbytes, dtype=torch.uint8, device="cuda") for _ in range(count)]
    return any(t.data_ptr() < ptr + nbytes and ptr < t.data_ptr() + nbytes for t in fresh)


def test_dropped_bias_list_stays_until_its_reader_is_done(cuda_lib):
    """A list made on one stream, read on another and dropped at once: its memory is not handed out meanwhile."""
    from nova_b200.logits import LogitBias, adjust_logits

    rows, v = 16, 50257
    entries = [{(37 * i + 11 * r) % v: 0.5 * i - 3.0 for i in range(200)} for r in range(rows)]
    x = torch.zeros(rows, v, dtype=torch.float32, device="cuda")
    want = torch.zeros(rows, v)
    for r, e in enumerate(entries):
        for t, w in e.items():
            want[r, t] = w
    adjust_logits(x, bias=LogitBias(entries, v))              # loads the kernel
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    bias = LogitBias(entries, v)
    ptr, nbytes = bias.buffer.data_ptr(), bias.buffer.numel() * 4
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        out = adjust_logits(x, bias=bias)
    del bias
    assert not others_memory(ptr, nbytes)
    side.synchronize()
    assert torch.equal(out.cpu(), want)


def test_plans_stay_until_their_reader_is_done(cuda_lib):
    """The same for the buffers of attention and adapter plans."""
    from nova_b200.lora import LoraPlan, lora_add
    from nova_b200.paged import paged_attention

    s = ref.State([1, 90], [3000, 150], 2, 8, seed=9)
    want, bound, _, _ = ref.attention(s)
    cache, q = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda()), s.q.cuda()
    g = torch.Generator().manual_seed(2)
    x, base = torch.randn(900, 64, generator=g).half().cuda(), torch.randn(900, 64, generator=g).half().cuda()
    a, b = torch.randn(1, 8, 64, generator=g).half().cuda(), torch.randn(1, 64, 8, generator=g).half().cuda()
    attend = lambda p: paged_attention(q, *cache, p)          # noqa: E731
    adapt = lambda p: lora_add(x, base, a, b, p)              # noqa: E731
    for make, use in ((s.plan, attend), (lambda: LoraPlan([900], [0], [8]), adapt)):
        expected = use(make())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        plan = make()
        held = [(t.data_ptr(), t.numel() * t.element_size()) for t in (plan.buffer, plan.workspace) if t.numel()]
        torch.cuda.synchronize()                              # the workspace is zeroed on the plan's own stream
        with torch.cuda.stream(side):
            torch.cuda._sleep(LONG)
            out = use(plan)
        del plan
        assert not any(others_memory(*h, count=8) for h in held)
        side.synchronize()
        assert torch.equal(out, expected)


def test_bias_of_another_kind_is_refused(cuda_lib):
    import copy

    from nova_b200.logits import LogitBias, adjust_logits

    x = torch.zeros(2, 100, dtype=torch.float16, device="cuda")
    for bad in (ref.State([1], [70], 1, 1).plan(), LogitBias([{1: 2.0}, {}], 100, device="cpu"), LogitBias([{}], 100)):
        with pytest.raises(ValueError):
            adjust_logits(x, bias=bad)
    bias = LogitBias([{1: 2.0}, {5: -1.0}], 100)
    other = copy.deepcopy(bias)                               # a copy reads its own memory
    assert other._handle[4].data_ptr() == other.buffer.data_ptr() != bias.buffer.data_ptr()
    assert torch.equal(adjust_logits(x, bias=other), adjust_logits(x, bias=bias))

"""A plan reaches the compiled binding by a handle that only its own kind of call
takes.  Nothing here launches: every call is refused on the host."""

from __future__ import annotations

import copy
import ctypes

import pytest
import torch

from nova_b200 import _lib
from nova_b200.lora import lora_add
from nova_b200.paged import paged_attention, paged_read, qkv_append

T = torch.zeros(1, 8, 128, dtype=torch.float16)


class Plan:
    """A plan's handle over fields of zeros: nothing in them may be followed before its kind is known."""

    def __init__(self, name, handle=None):
        self._fields = (ctypes.c_int64 * 10)()
        self._handle = _lib.handle(self._fields, name) if handle is None else handle


CALLS = {
    "attention": (_lib.LORA_PLAN, lambda p: paged_attention(T, T, T, T, p)),
    "append": (_lib.LORA_PLAN, lambda p: qkv_append(T, T, T, T, p)),
    "read": (_lib.LORA_PLAN, lambda p: paged_read(T, T, T, p)),
    "lora": (_lib.PAGE_PLAN, lambda p: lora_add(T, T, T, T, p)),
}


@pytest.mark.parametrize("call", CALLS)
def test_a_plan_of_another_kind_is_refused(call):
    other, run = CALLS[call]
    for plan in (Plan(other), Plan(b"another"), Plan(b"", handle="text"), Plan(b"", handle=(1, 2)), Plan(b"", handle=None)):
        with pytest.raises(ValueError, match="must be a nova_b200"):
            run(plan)
    for number in (0, 64):                    # a number is no address: 0 marks a plan on the host
        with pytest.raises(ValueError, match="not on a CUDA device"):
            run(Plan(b"", handle=number))


def test_a_handle_is_not_copied():
    plan = Plan(_lib.PAGE_PLAN)
    assert copy.copy(plan)._handle is plan._handle            # a shallow copy keeps the fields alive
    with pytest.raises(TypeError):
        copy.deepcopy(plan)


@pytest.mark.gpu
def test_real_plans_are_told_apart(cuda_lib):
    from nova_b200.lora import LoraPlan
    from paged_reference import State

    s = State([1], [70], 1, 1)
    pages, adapters = s.plan(), LoraPlan([1], [0], [8])
    with pytest.raises(ValueError, match="must be a nova_b200.PagePlan"):
        paged_attention(s.q.cuda(), s.codes.cuda(), s.scales.cuda(), s.tails.cuda(), adapters)
    x = torch.zeros(1, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="must be a nova_b200.LoraPlan"):
        lora_add(x, x, torch.zeros(1, 8, 64, dtype=torch.float16, device="cuda"),
                 torch.zeros(1, 64, 8, dtype=torch.float16, device="cuda"), pages)
    for plan in (pages, adapters):
        with pytest.raises(TypeError):
            copy.deepcopy(plan)

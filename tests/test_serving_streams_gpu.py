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

"""GPU: token history whose offsets name more than the tokens.  The tokens are a
piece of a larger tensor, so that every number the offsets could reach is memory
of the test's own."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompt", [True, False])
@pytest.mark.parametrize("offsets", [
    [0, 4, 900, 900],            # the second row ends past the tokens
    [0, 700, 900, 950],          # every row does
    [-50, 4, 7, 10],             # a row begins before them
    [10, 4, 7, 2],               # rows that end before they begin
    [0, 10, 10, 10],
])
def test_offsets_past_the_tokens_are_not_followed(cuda_lib, prompt, offsets):
    from nova_b200.logits import add_generated, add_prompt, new_history

    around = torch.arange(1000, device="cuda") % 64 + 100     # what may not be entered
    tokens = around[100:110]
    tokens.copy_(torch.tensor([1, 2, 3, 4, 5, 5, 7, 8, 9, 9]))
    h = new_history(3, 200)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    (add_prompt if prompt else add_generated)(h, tokens, off)
    want = torch.zeros(3, 200, dtype=torch.long)
    for r in range(3):
        for t in tokens[max(offsets[r], 0):max(0, min(offsets[r + 1], 10))].tolist():
            want[r, t] = -32768 if prompt else want[r, t] + 1
    assert torch.equal(h.cpu().long(), want)

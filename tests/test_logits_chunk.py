"""CPU: the bias lists are built by the chunk that the C interface names."""

from __future__ import annotations

import re

from conftest import REPO
from nova_b200 import logits


def test_chunk_is_the_headers():
    header = (REPO / "include" / "nova_b200.h").read_text()
    assert int(re.search(r"#define NOVA_LOGITS_CHUNK (\d+)", header).group(1)) == logits.CHUNK


def test_lists_by_chunk():
    c = logits.CHUNK
    bias = logits.LogitBias([{0: 1.0, c - 1: 2.0, c: 3.0}, {}, {2 * c: 4.0}], 2 * c + 1, device="cpu")
    assert bias.off.tolist() == [0, 2, 3, 3, 3, 3, 3, 3, 3, 4]
    assert bias.token.tolist() == [0, c - 1, c, 2 * c] and bias.value.tolist() == [1.0, 2.0, 3.0, 4.0]

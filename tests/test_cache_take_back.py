"""CPU: the paged cache's bookkeeping when a planned step is taken back."""

from __future__ import annotations

import random

import pytest

from nova_b200.paged import PAGE, PagedKVCache


def state(c):
    return list(c._free), {i: (r["slot"], r["flip"], r["length"], list(r["pages"])) for i, r in c._requests.items()}


def test_a_step_taken_back_leaves_no_trace():
    rng = random.Random(1)
    c = PagedKVCache(1, 1, 1, num_pages=40, max_requests=3, device="cpu")
    ids = [c.add() for _ in range(3)]
    for _ in range(60):
        step = rng.sample(ids, rng.randint(1, 3))
        new = [rng.choice([0, 1, 5, 64, rng.randint(0, 150)]) for _ in step]
        before = state(c)
        try:
            plan = c.plan(step, new)
        except RuntimeError:                                  # out of pages: nothing has changed
            assert state(c) == before
            c.release(ids[0])
            ids[0] = c.add()
            continue
        if rng.random() < 0.5:
            c.take_back(plan)
            assert state(c) == before
            again = c.plan(step, new)                         # the same step once more: the same plan
            assert (again.host == plan.host).all() and again.tail_out == plan.tail_out
        else:
            assert all(c.length(i) == before[1][i][2] + n for i, n in zip(step, new))


def test_only_the_latest_plan_is_taken_back():
    c = PagedKVCache(1, 1, 1, num_pages=8, max_requests=2, device="cpu")
    a, b = c.add(), c.add()
    first = c.plan([a, b], [PAGE, 3])
    second = c.plan([b], [1])
    before = state(c)
    with pytest.raises(ValueError, match="planned again"):
        c.take_back(first)
    assert state(c) == before
    c.take_back(second)
    with pytest.raises(ValueError, match="taken back already"):
        c.take_back(second)
    with pytest.raises(ValueError, match="planned again"):    # b has its list of pages from before again, a too
        c.release(a)
        c.take_back(first)
    assert c.length(b) == 3

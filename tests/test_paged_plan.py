"""CPU: the plan of a paged step -- records, work lists covering every query row
and block exactly once, and the refusals -- built without a GPU."""

from __future__ import annotations

import numpy as np
import pytest

from nova_b200.paged import PagedKVCache, PagePlan

PAGE = 64


def make(q, kv, hq=8, hkv=2, **kw):
    pages, at = [], 0
    for n in kv:
        pages.append(list(range(at, at + n // PAGE)))
        at += n // PAGE
    tin = [2 * i for i in range(len(q))]
    tout = [2 * i + (n // PAGE != (n - m) // PAGE) for i, (m, n) in enumerate(zip(q, kv))]
    kw = {"tail_in": tin, "tail_out": tout, "num_q_heads": hq, "num_kv_heads": hkv, "device": "cpu", **kw}
    return PagePlan(q, kv, kw.pop("pages", pages), **kw)


def rows_items(plan, w=0):
    return np.concatenate([plan.host[r.off:r.off + 16 * r.n].reshape(-1, 16) for r in plan.info.sched[w].rows])


def test_records_and_lists():
    p = make([5, 1, 0, 100], [5, 130, 64, 300])
    i = p.info
    seqs = p.host[i.seq_off:i.seq_off + 32].reshape(4, 8)
    assert seqs[:, 0].tolist() == [0, 5, 6, 6] and seqs[:, 2].tolist() == [5, 130, 64, 300]
    assert p.tokens == 106
    assert p.host[i.pos_off:i.pos_off + 106].tolist() == [*range(5), 129, *range(200, 300)]
    open_tokens = p.host[i.open_off:i.open_off + 4 * i.n_open].reshape(-1, 4)       # row, position, tail buffer
    assert open_tokens[:, :3].tolist() == ([[t, t, 0] for t in range(5)] + [[5, 129, 2]]
                                           + [[6 + t - 200, t, 7] for t in range(256, 300)])
    write = p.host[i.write_off:i.write_off + 8 * i.n_write].reshape(-1, 8)
    # pages that fill: block, first new position, length, its token row, tail before and after, page
    assert write[:, :7].tolist() == [[3, 200, 300, 6, 6, 7, 6]]
    assert p.read_rows == 5 + 2 + 0 + (300 - 192)


def test_read_from():
    p = make([1, 1, 1], [200, 70, 1], read_from=[0, 70, 0])
    i = p.info
    read = p.host[i.read_off:i.read_off + 8 * i.n_read].reshape(-1, 8)
    assert p.read_rows == 201
    # block, first copied position, length, its output row
    assert read[:, :4].tolist() == [[0, 0, 200, 0], [1, 0, 200, 0], [2, 0, 200, 0], [3, 0, 200, 0], [0, 0, 1, 200]]
    p = make([1], [200], read_from=[100])
    read = p.host[p.info.read_off:p.info.read_off + 8 * p.info.n_read].reshape(-1, 8)
    assert p.read_rows == 100
    assert read[:, :4].tolist() == [[1, 100, 200, 0], [2, 100, 200, 0], [3, 100, 200, 0]]


@pytest.mark.parametrize("window", [0, 1, 63, 200])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (6, 2), (16, 1)])
def test_every_row_sees_its_blocks_once(hq, hkv, window):
    """For each query row (and KV head): the blocks of all work items and
    segments that hold it are its key range's blocks (or more of the same
    tile's), each once; a cut tile's partials are joined in order."""
    q, kv = [1, 3, 0, 17, 1, 1], [1, 64, 10, 400, 5000, 63]
    p = make(q, kv, hq, hkv, windows=(window,))
    gq = hq // hkv
    seen = {}
    at = {sum(q[:i]): i for i in range(len(q)) if q[i]}
    for row0, nrows, b0, b1, part0, split, n, q_start, start, kv_len, page_off, tail, *first in rows_items(p).tolist():
        seq = at[q_start]
        assert first == [page_off + b if b < min(b1, kv_len // PAGE) else -1 for b in range(b0, b0 + 4)]
        assert (q_start, start, kv_len) == (sum(q[:seq]), kv[seq] - q[seq], kv[seq])
        assert page_off == sum(n // PAGE for n in kv[:seq]) and (not kv_len % PAGE or tail == p.tail_out[seq])
        assert 0 <= split < n and (part0 < 0) == (n == 1) and b1 > b0 and nrows >= 1
        for r in range(row0, row0 + nrows):
            seen.setdefault((seq, r), []).extend(range(b0, b1))
    tiles = {}
    sched = p.info.sched[0]
    segs = p.host[sched.segs_off:sched.segs_off + 16 * sched.n_segs].reshape(-1, 16).tolist()
    assert sched.n_ctas <= 148
    order = []                                  # every CTA's segments, one CTA after another: the tiles in order
    for cta in range(sched.n_ctas):
        while cta >= 0:
            order.append(segs[cta])
            cta = segs[cta][15]
    assert len(order) == len(segs) and sorted(map(tuple, order)) == sorted(map(tuple, segs))
    for head, row0, nrows, b0, b1, part, q_start, start, kv_len, page_off, tail, *first in order:
        seq = at[q_start]
        assert (q_start, start, kv_len) == (sum(q[:seq]), kv[seq] - q[seq], kv[seq])
        assert page_off == sum(n // PAGE for n in kv[:seq]) and (not kv_len % PAGE or tail == p.tail_out[seq])
        assert first[:4] == [page_off + b if b < min(b1, kv_len // PAGE) else -1 for b in range(b0, b0 + 4)]
        assert b1 > b0 and 1 <= nrows <= 256
        tiles.setdefault((seq, head, row0, nrows), []).append((b0, b1, part))
    joins = p.host[sched.joins_off:sched.joins_off + 8 * sched.n_joins].reshape(-1, 8).tolist()
    joins = {tuple(j[:4]): (j[4], j[5]) for j in joins}
    for key, parts in tiles.items():
        assert [x[1] for x in parts[:-1]] == [x[0] for x in parts[1:]]
        if len(parts) > 1:
            first, count = joins.pop(key)
            assert [x[2] for x in parts] == list(range(first, first + count))
        else:
            assert parts[0][2] == -1
        seq, head, row0, nrows = key
        for r in range(row0, row0 + nrows):
            blocks = [b for b0, b1, _ in parts for b in range(b0, b1)]
            assert seen.setdefault((seq, r), blocks) == blocks    # every head the same
    assert not joins and len(tiles) % hkv == 0
    for i, (m, n) in enumerate(zip(q, kv)):
        for r in range(m * gq):
            pos = n - m + r // gq
            first = max(0, pos - window + 1) // PAGE if window else 0
            got = seen.pop((i, r))
            assert len(set(got)) == len(got)
            assert set(range(first, pos // PAGE + 1)) <= set(got) <= set(range((n - 1) // PAGE + 1))
    assert not seen


@pytest.mark.parametrize("change,message", [
    (dict(kv=[4, 130]), "new tokens and length"),
    (dict(q=[-1, 1]), "new tokens and length"),
    (dict(pages=[[], [3]]), "are needed"),
    (dict(pages=[[], [3, -4]]), "page"),
    (dict(tail_in=[0, 1], tail_out=[0, 3]), "must be tail_in"),
    (dict(tail_out=[0, 0], tail_in=[0, 0]), "share tail buffer"),
    (dict(tail_in=[0, -1], tail_out=[0, -1]), "needs a tail buffer"),
    (dict(q=[5, 70], kv=[5, 130], tail_in=[0, 2], tail_out=[0, 2]), "must differ"),
    (dict(q=[70, 70], kv=[70, 70], pages=[[0], [0]]), "written twice"),
    (dict(hq=7), "multiple of kv_heads"),
    (dict(windows=(-1,)), "window"),
    (dict(windows=(0, 0)), "different"),
    (dict(windows=(0, 1, 2, 3, 4)), "at most"),
    (dict(read_from=[0, 131]), "read_from"),
    (dict(read_from=[0]), "one position"),
    (dict(pages=[[]]), "same requests"),
])
def test_refusals(change, message):
    kw = {"q": [5, 1], "kv": [5, 130], **change}
    with pytest.raises(ValueError, match=message):
        make(kw.pop("q"), kw.pop("kv"), **kw)


def test_shared_prefix_pages_are_allowed():
    """Two requests may read the same full pages; only pages that the step writes must be their own."""
    make([1, 1], [130, 140], pages=[[0, 1], [0, 1]])


def test_cache_hands_out_pages_and_tails():
    c = PagedKVCache(1, 2, 4, num_pages=6, max_requests=2, device="cpu")
    a, b = c.add(), c.add()
    with pytest.raises(RuntimeError, match="slot"):
        c.add()
    p = c.plan([a, b], [130, 10])
    assert c.length(a) == 130 and c.free_pages() == 4
    out = p.tail_out
    p = c.plan([b, a], [54, 1])            # b fills its page, a's stays open
    assert c.free_pages() == 3 and p.kv_lens == [64, 131]
    assert p.tail_out[1] == out[0]
    with pytest.raises(RuntimeError, match="pages"):
        c.plan([a], [1000])
    assert c.length(a) == 131 and c.free_pages() == 3
    with pytest.raises(ValueError):
        c.plan([a, a], [1, 1])
    with pytest.raises(ValueError):
        c.plan([a], [-1])
    used = {x for r in c._requests.values() for x in r["pages"]}
    assert len(used) == 3 and not used & set(c._free)
    c.release(a)
    assert c.free_pages() == 5
    c.add()


def test_tail_alternates_when_a_page_opens():
    c = PagedKVCache(1, 1, 1, num_pages=64, max_requests=1, device="cpu")
    r = c.add()
    prev, rng = None, np.random.default_rng(0)
    for n in rng.integers(0, 150, 30).tolist():
        start = c.length(r)
        if (start + n) // PAGE - start // PAGE > c.free_pages():
            break
        p = c.plan([r], [n])
        if prev is not None and start % PAGE:
            tin = int(p.host[p.info.seq_off + 4])
            assert tin == prev
            if (start + n) % PAGE:
                assert (p.tail_out[0] == tin) == ((start + n) // PAGE == start // PAGE)
        prev = p.tail_out[0]


def test_binding_refuses_without_a_gpu():
    """The compiled binding loads on the CPU and refuses host plans and other objects before anything else."""
    import torch

    from nova_b200 import _lib
    from nova_b200.logits import adjust_logits
    from nova_b200.lora import LoraPlan, lora_add
    from nova_b200.paged import paged_attention, paged_read

    assert _lib.fast().__name__.endswith("_fast")
    p, t = make([1], [1]), torch.zeros(1, 8, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="plan is not on a CUDA device"):
        paged_attention(t, t, t, t, p)
    with pytest.raises(ValueError, match="plan is not on a CUDA device"):
        paged_read(t, t, t, p)
    with pytest.raises(ValueError, match="plan is not on a CUDA device"):
        lora_add(t, t, t, t, LoraPlan([1], [0], [8], device="cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        adjust_logits(t[0])
    with pytest.raises(ValueError, match="tensor"):
        adjust_logits(None)
    with pytest.raises(AttributeError):
        paged_read(t, t, t, object())
    with pytest.raises(TypeError):
        _lib.fast().paged_read(t, t)

"""Low-rank adapters of many requests (nova_lora_add) against the formula in 64
bits, and the host-side plan (CPU).

Bound: the first product is an fp32 sum of k exact products (k * 2^-24 of the
sum of magnitudes), scaled and rounded to fp16 once (2^-11; 2^-25 below the
normal range), the second one an fp32 sum over the rank, and the result is
rounded once."""

from __future__ import annotations

import numpy as np
import pytest
import torch


def make(tokens, which, ranks, k, n, r, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = sum(tokens)
    x = torch.randn(t, k, generator=g).half()
    base = torch.randn(t, n, generator=g).half()
    a = (torch.randn(len(ranks), r, k, generator=g) * k ** -0.5).half()
    b = (torch.randn(len(ranks), n, r, generator=g) * 0.3).half()
    scaling = 0.5 + torch.rand(len(ranks), generator=g)
    return x, base, a, b, scaling


def reference(x, base, a, b, scaling, tokens, which, ranks):
    out, err = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64)
    t0 = 0
    for m, w in zip(tokens, which):
        rows = slice(t0, t0 + m)
        t0 += m
        if w < 0 or not m:
            continue
        r = ranks[w]
        s = float(scaling[w])
        xa, aa, bb = x[rows].double(), a[w, :r].double(), b[w, :, :r].double()
        h, size = xa @ aa.t() * s, xa.abs() @ aa.abs().t() * s
        eh = x.shape[1] * 2.0 ** -24 * size + 2.0 ** -11 * h.abs() + 2.0 ** -25
        out[rows] += h @ bb.t()
        err[rows] = eh @ bb.abs().t() + (r + 2) * 2.0 ** -24 * (h.abs() @ bb.abs().t() + base[rows].abs())
    return out, err + 2.0 ** -11 * (out.abs() + err) + 2.0 ** -25


CASES = [
    # tokens, adapter of each request, ranks, k, n, max_rank
    ([1], [0], [8], 64, 32, 8),
    ([1], [0], [1], 8, 8, 8),
    ([1, 1, 1], [2, -1, 0], [16, 3, 9], 2560, 1024, 16),
    ([1] * 40, [i % 7 - 1 for i in range(40)], [16, 16, 5, 12, 16, 8], 2560, 6144, 16),
    ([17, 0, 3], [0, 0, 1], [32, 30], 200, 72, 32),
    ([70, 1, 130, 5], [1, 0, 1, -1], [64, 50], 1024, 328, 64),
    ([33, 100], [0, 1], [128, 77], 776, 200, 128),
    ([5, 90], [0, -1], [7], 4096, 2560, 16),
    ([300], [3], [8, 8, 8, 31], 264, 96, 40),
    ([900, 77, 300], [0, 1, 2], [16, 9, 64], 136, 328, 64),
    ([1000, 60], [0, 1], [128, 100], 96, 40, 128),
    ([1030, 1], [1, 0], [8, 13], 72, 64, 16),
    ([1100], [0], [30], 40, 104, 32),
    ([64, 64], [0, 1], [0, 16], 512, 256, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,which,ranks,k,n,r", CASES)
def test_matches_formula(cuda_lib, tokens, which, ranks, k, n, r):
    from nova_b200.lora import LoraPlan, lora_add

    x, base, a, b, scaling = make(tokens, which, ranks, k, n, r)
    for i, rank in enumerate(ranks):          # entries past a rank are never used
        a[i, rank:] = float("nan")
        b[i, :, rank:] = float("inf")
    want, bound = reference(x, base, a, b, scaling, tokens, which, ranks)
    plan = LoraPlan(tokens, which, ranks)
    dev = [t.cuda() for t in (x, base, a, b)]
    got = lora_add(*dev, plan, scaling=scaling.cuda())
    d = (got.double().cpu() - want).abs()
    assert (d <= bound).all(), f"{(d > bound).sum()} beyond the bound (max {d.max():.3e})"
    assert torch.equal(dev[1].cpu(), base)
    # in place, and from and into padded rows: the same bits
    wide_x = torch.full((x.shape[0], k + 8), float("nan"), dtype=torch.float16, device="cuda")
    wide_x[:, :k] = dev[0]
    wide = torch.full((x.shape[0], n + 24), 5.0, dtype=torch.float16, device="cuda")
    wide[:, :n] = dev[1]
    out = lora_add(wide_x[:, :k], wide[:, :n], dev[2], dev[3], plan, scaling=scaling.cuda(), out=wide[:, :n])
    assert torch.equal(out, got) and (wide[:, n:] == 5.0).all()


@pytest.mark.gpu
def test_without_scaling_and_without_adapters(cuda_lib):
    from nova_b200.lora import LoraPlan, lora_add

    x, base, a, b, _ = make([3, 4], [0, 0], [8], 128, 64, 8)
    want, bound = reference(x, base, a, b, torch.ones(1), [3, 4], [0, 0], [8])
    dev = [t.cuda() for t in (x, base, a, b)]
    got = lora_add(*dev, LoraPlan([3, 4], [0, 0], [8]))
    assert ((got.double().cpu() - want).abs() <= bound).all()
    got = lora_add(*dev, LoraPlan([3, 4], [-1, -5], [8]))
    assert torch.equal(got.cpu(), base)
    got = lora_add(*dev, LoraPlan([7], [-1], [8]), out=dev[1])
    assert torch.equal(got.cpu(), base)


@pytest.mark.gpu
def test_refusals(cuda_lib):
    from nova_b200.lora import LoraPlan, lora_add

    x, base, a, b, s = (t.cuda() for t in make([4], [0], [8], 64, 32, 8))
    plan = LoraPlan([4], [0], [8])
    bad = [
        lambda: lora_add(x.float(), base, a, b, plan),
        lambda: lora_add(x.cpu(), base, a, b, plan),
        lambda: lora_add(x[:3], base[:3], a, b, plan),
        lambda: lora_add(x, base, a, b[:, :, :4], plan),
        lambda: lora_add(x, base, a[:, :4].contiguous(), b[:, :, :4].contiguous(), plan),       # below the plan's rank
        lambda: lora_add(x[:, :60].contiguous(), base, a[:, :, :60].contiguous(), b, plan),     # K % 8
        lambda: lora_add(x, base, a, b, plan, scaling=s.half()),
        lambda: lora_add(x, base, a, b, plan, out=base.float()),
        lambda: lora_add(x, base, a.transpose(1, 2), b, plan),
        lambda: lora_add(torch.zeros(4, 65, dtype=torch.float16, device="cuda")[:, 1:], base, a, b, plan),  # alignment
        lambda: lora_add(x, base, a, b, LoraPlan([4], [0], [8, 8])),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")


def test_plan_gathers_rows_by_adapter():
    from nova_b200.lora import LoraPlan

    tokens, which, ranks = [3, 1, 0, 40, 2], [1, -1, 0, 0, 1], [4, 16, 9]
    p = LoraPlan(tokens, which, ranks, device="cpu")
    tiles = p.buffer.view(p.n_tiles, 4 + p.tile_rows).tolist()
    of_row = np.repeat(which, tokens).tolist()
    rows = [r for t in tiles for r in t[4:4 + t[2]]]
    assert sorted(rows) == list(range(46)) and p.tile_rows == 16 and p.max_rank == 16
    for adapter, rank, n, zero, *mine in tiles:
        assert 1 <= n <= p.tile_rows and rank == (ranks[adapter] if adapter >= 0 else 0) and zero == 0
        assert all(of_row[r] == adapter for r in mine[:n]) and all(r == -1 for r in mine[n:])
    assert LoraPlan([1] * 40, [0] * 20 + [1] * 20, [8, 8], device="cpu").tile_rows == 16
    assert LoraPlan([700, 500], [0, 1], [8, 8], device="cpu").tile_rows == 64
    assert LoraPlan([1] * 64, list(range(64)), [8] * 64, device="cpu").tile_rows == 16


@pytest.mark.parametrize("args,message", [
    (([1], [0, 1], [8]), "one length"),
    (([-1], [0], [8]), "negative"),
    (([1], [1], [8]), "adapter 1 of 1"),
    (([1], [0], [129]), "ranks"),
    (([1], [0], [-1]), "ranks"),
])
def test_plan_refusals(args, message):
    from nova_b200.lora import LoraPlan

    with pytest.raises(ValueError, match=message):
        LoraPlan(*args, device="cpu")

"""Low-rank adapters whose first product or scaling is far from one, against the
formula in 64 bits.

Bound: h = x A^T is an fp32 sum of k exact products (k * 2^-24 of the sum of
magnitudes); each row is rounded to fp16 at a power of two that puts its largest
entry at 2^14 or more, so an entry is off by 2^-11 of itself, or, below the
normal range, by 2^-25 * 2^-14 of the row's largest; the second product is an
fp32 sum over the rank with the factor and base (r + 3 roundings), and the
result is rounded once."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def formula(x, base, a, b, s, rank):
    xa, aa, bb = x.double(), a[0, :rank].double(), b[0, :, :rank].double()
    s = float(torch.tensor(s, dtype=torch.float32))
    h, size = xa @ aa.t(), xa.abs() @ aa.abs().t()
    eh = x.shape[1] * 2.0 ** -24 * size + 2.0 ** -11 * h.abs() + 2.0 ** -39 * h.abs().amax(1, keepdim=True)
    want = base.double() + s * (h @ bb.t())
    err = abs(s) * (eh @ bb.abs().t()) + (rank + 3) * 2.0 ** -24 * (abs(s) * (h.abs() @ bb.abs().t()) + base.double().abs())
    return want, err + 2.0 ** -11 * (want.abs() + err) + 2.0 ** -25


SIZES = {                        # spread of x, A and B, and the scaling
    "product past fp16": (200.0, 100.0, 2e-4, 0.01),
    "scaling past fp16": (10.0, 0.5, 1e-4, 2e4),
    "tiny scaling, large B": (1.0, 0.05, 3e3, 1e-6),
    "tiny product": (1e-3, 1e-3, 2e3, 50.0),
    "negative scaling": (30.0, 30.0, 1e-3, -0.5),
}


@pytest.mark.parametrize("tokens", [3, 700])           # one launch, two launches
@pytest.mark.parametrize("rank,r", [(3, 8), (16, 16), (30, 32), (64, 64), (128, 128)])
@pytest.mark.parametrize("sizes", SIZES)
def test_any_size_of_the_first_product(cuda_lib, sizes, rank, r, tokens):
    from nova_b200.lora import LoraPlan, lora_add

    sx, sa, sb, s = SIZES[sizes]
    k, n = 520, 136
    g = torch.Generator().manual_seed(rank + tokens)
    x = (torch.randn(tokens, k, generator=g) * sx).half()
    x *= (2.0 ** torch.randint(-6, 3, (tokens, 1), generator=g)).half()      # rows of one tile differ
    x[1] = 0
    a, b = (torch.randn(1, r, k, generator=g) * sa).half(), (torch.randn(1, n, r, generator=g) * sb).half()
    b[0, :8] = 0                                                             # columns that the adapter leaves alone
    b[0, 8:16, 1::2], a[0, 1::2] = -b[0, 8:16, ::2], a[0, ::2] * 1.001       # and terms that nearly cancel
    base = torch.randn(tokens, n, generator=g).half()
    want, bound = formula(x, base, a, b, s, rank)
    got = lora_add(x.cuda(), base.cuda(), a.cuda(), b.cuda(), LoraPlan([tokens], [0], [rank]),
                   scaling=torch.tensor([s], device="cuda")).double().cpu()
    fits = want.abs() + bound < 65504                                        # what fp16 can hold
    assert fits.float().mean() > 0.99 and torch.isfinite(got[fits]).all()
    d = (got - want).abs()[fits]
    assert (d <= bound[fits]).all(), f"{(d > bound[fits]).sum()} beyond the bound (max {d.max():.3e})"
    assert torch.equal(got[:, :8], base[:, :8].double()) and torch.equal(got[1], base[1].double())


@pytest.mark.parametrize("tokens", [5, 700])
def test_a_row_that_is_not_finite_stays_alone(cuda_lib, tokens):
    from nova_b200.lora import LoraPlan, lora_add

    g = torch.Generator().manual_seed(8)
    x, base = torch.randn(tokens, 64, generator=g).half(), torch.randn(tokens, 32, generator=g).half()
    a, b = torch.randn(1, 8, 64, generator=g).half(), torch.randn(1, 32, 8, generator=g).half()
    args = (base.cuda(), a.cuda(), b.cuda(), LoraPlan([tokens], [0], [8]))
    clean = lora_add(x.cuda(), *args)
    x[2, 5], x[4, 7] = float("inf"), float("nan")
    got = lora_add(x.cuda(), *args)
    assert not torch.isfinite(got[2]).any() and torch.isnan(got[4]).all()
    rest = [i for i in range(tokens) if i not in (2, 4)]
    assert torch.equal(got[rest], clean[rest])


def test_a_row_does_not_depend_on_its_tile(cuda_lib):
    """The power of two is the row's own: other rows of the batch change nothing."""
    from nova_b200.lora import LoraPlan, lora_add

    g = torch.Generator().manual_seed(9)
    x, base = torch.randn(16, 256, generator=g).half().cuda(), torch.randn(16, 64, generator=g).half().cuda()
    a, b = torch.randn(1, 16, 256, generator=g).half().cuda(), torch.randn(1, 64, 16, generator=g).half().cuda()
    together = lora_add(x, base, a, b, LoraPlan([16], [0], [16]))
    x2 = x.clone()
    x2[1:] *= 100.0
    assert torch.equal(lora_add(x2, base, a, b, LoraPlan([16], [0], [16]))[0], together[0])

"""Per-request logit controls against the formula in 64 bits.

Bound: four fp32 operations (2^-22 of the magnitudes in all) and one rounding to
the logits' type."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, hist, rep, freq, pres, entries, allowed, which):
    """(values, magnitudes of the terms) in 64 bits."""
    rows, v = x.shape
    y = x.double()
    size = torch.zeros_like(y)
    if hist is not None:
        h = hist.long()
        times = torch.where(h < 0, h + 32768, h)
        r = torch.ones(rows, 1, dtype=torch.float64) if rep is None else rep.double()[:, None]
        y = torch.where(h != 0, torch.where(y > 0, y / r, y * r), y)
        f = 0.0 if freq is None else freq.double()[:, None] * times
        p = 0.0 if pres is None else pres.double()[:, None] * (times > 0)
        size = y.abs() + f + p
        y = y - f - p
    for i, e in enumerate(entries or []):
        for t, w in e.items():
            w = float(torch.tensor(w, dtype=torch.float32))
            y[i, t] += w
            size[i, t] += abs(w)
    if allowed is not None:
        for i in range(rows):
            m = i if which is None else int(which[i])
            if m >= 0:
                bits = (((allowed[m].long() & 0xFFFFFFFF)[:, None] >> torch.arange(32)) & 1).flatten()[:v]
                y[i, bits == 0] = -math.inf
    return y, size


def make(rows, v, dtype, seed=0, masks=0, biases=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, v, generator=g) * 4).to(dtype)
    hist = torch.where(torch.rand(rows, v, generator=g) < 0.05, torch.randint(0, 9, (rows, v), generator=g), 0)
    hist = hist + torch.where(torch.rand(rows, v, generator=g) < 0.05, -32768, 0)
    hist[:, 0], hist[:, -1] = 32767, -1       # count at its end, with and without the prompt bit
    rep, freq, pres = 1 + torch.rand(rows, generator=g), torch.rand(rows, generator=g), torch.rand(rows, generator=g)
    freq *= 0.01
    entries = [{int(t): float(w) for t, w in zip(torch.randint(0, v, (biases,), generator=g),
                                                 torch.randn(biases, generator=g) * 5)} for _ in range(rows)]
    allowed = torch.randint(-2 ** 31, 2 ** 31, (max(masks, 1), -(-v // 32)), generator=g).to(torch.int32)
    return x, hist.to(torch.int16), rep, freq, pres, entries, allowed


def check(got, want, size, dtype):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want) & ~torch.isnan(want)
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    bound = (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24) * want[ok].abs() + 2.0 ** -22 * size[ok] + 2.0 ** -25
    d = (got[ok] - want[ok]).abs()
    assert (d <= bound).all(), f"{(d > bound).sum()} beyond the bound (max {d.max():.3e})"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,v", [(1, 1), (1, 7), (3, 33), (2, 2048), (5, 2049), (4, 4097), (3, 50257), (2, 151936)])
def test_matches_formula(cuda_lib, rows, v, dtype):
    from nova_b200.logits import LogitBias, adjust_logits

    x, hist, rep, freq, pres, entries, allowed = make(rows, v, dtype, seed=v, masks=3, biases=min(v, 60))
    which = torch.tensor([(-1, 2, 0, 1)[i % 4] for i in range(rows)], dtype=torch.int32)
    want, size = reference(x, hist, rep, freq, pres, entries, allowed, which)
    bias = LogitBias(entries, v)
    dev = {"history": hist.cuda(), "repetition": rep.cuda(), "frequency": freq.cuda(), "presence": pres.cuda(),
           "bias": bias, "allowed": allowed.cuda(), "allowed_row": which.cuda()}
    got = adjust_logits(x.cuda(), **dev)
    check(got, want, size, dtype)
    # in place, in padded rows of another alignment for each tensor: the same bits
    wide = torch.full((rows, v + 13), 3.0, dtype=dtype, device="cuda")
    wide[:, 5:5 + v] = x.cuda()
    dev["history"] = torch.zeros(rows, v + 3, dtype=torch.int16, device="cuda")
    dev["history"][:, 2:2 + v] = hist.cuda()
    dev["history"] = dev["history"][:, 2:2 + v]
    out = adjust_logits(wide[:, 5:5 + v], out=wide[:, 5:5 + v], **dev)
    assert torch.equal(out, got) and (wide[:, :5] == 3.0).all() and (wide[:, 5 + v:] == 3.0).all()


@pytest.mark.parametrize("drop", ["history", "bias", "allowed", "repetition", "frequency", "presence", "all"])
def test_controls_are_optional(cuda_lib, drop):
    from nova_b200.logits import LogitBias, adjust_logits

    x, hist, rep, freq, pres, entries, allowed = make(3, 5000, torch.float16, masks=3, biases=9)
    args = {"history": hist, "repetition": rep, "frequency": freq, "presence": pres, "entries": entries, "allowed": allowed}
    for name in {"history": ("history", "repetition", "frequency", "presence"), "bias": ("entries",),
                 "all": tuple(args)}.get(drop, (drop,)):
        args[name] = None
    want, size = reference(x, args["history"], args["repetition"], args["frequency"], args["presence"], args["entries"],
                           args["allowed"], None)
    dev = {k: v.cuda() for k, v in args.items() if v is not None and k != "entries"}
    if args["entries"]:
        dev["bias"] = LogitBias(entries, 5000)
    check(adjust_logits(x.cuda(), **dev), want, size, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("lead,v,biases", [(0, 4096, 1500), (5, 6001, 4000), (7, 2050, 900), (1, 2047, 300)])
def test_many_biases_in_place(cuda_lib, lead, v, biases, dtype):
    """Bias lists longer than a CTA has threads; rows that begin inside a vector, where a CTA's tokens
    lie in two lists; the result written over the logits by whole vectors."""
    from nova_b200.logits import LogitBias, adjust_logits

    rows, width = 3, -(-(v + lead) // 8) * 8
    x, hist, rep, freq, pres, entries, allowed = make(rows, v, dtype, seed=v, masks=rows, biases=biases)
    want, size = reference(x, hist, rep, freq, pres, entries, allowed, None)
    logits = torch.full((rows, width), 3.0, dtype=dtype, device="cuda")
    history = torch.zeros(rows, width, dtype=torch.int16, device="cuda")
    logits[:, lead:lead + v], history[:, lead:lead + v] = x.cuda(), hist.cuda()
    out = logits[:, lead:lead + v]
    adjust_logits(out, history=history[:, lead:lead + v], repetition=rep.cuda(), frequency=freq.cuda(),
                  presence=pres.cuda(), bias=LogitBias(entries, v), allowed=allowed.cuda(), out=out)
    check(out, want, size, dtype)
    assert (logits[:, :lead] == 3.0).all() and (logits[:, lead + v:] == 3.0).all()


def test_masks_override_everything(cuda_lib):
    """NaN, infinities and the type's lowest value in masked places; a mask that leaves nothing; a
    mask number past the masks."""
    from nova_b200.logits import adjust_logits

    v = 100
    x = torch.zeros(4, v, dtype=torch.float16)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = math.nan, math.inf, -math.inf, torch.finfo(torch.float16).min
    allowed = torch.zeros(2, 4, dtype=torch.int32)
    allowed[1, 0] = 0b11 << 3
    which = torch.tensor([0, 1, -1, 2], dtype=torch.int32)
    got = adjust_logits(x.cuda(), allowed=allowed.cuda(), allowed_row=which.cuda()).cpu()
    assert (got[0] == -math.inf).all() and (got[3] == -math.inf).all()
    assert got[1, 3] == torch.finfo(torch.float16).min and got[1, 4] == 0
    assert (got[1, :3] == -math.inf).all() and (got[1, 5:] == -math.inf).all()
    assert torch.equal(got[2].nan_to_num(7.0), x[2].nan_to_num(7.0))


def test_history_counts(cuda_lib):
    from nova_b200.logits import add_generated, add_prompt, new_history

    rows, v = 5, 1001
    h = new_history(rows, v)
    g = torch.Generator().manual_seed(1)
    lens = [0, 1, 700, 3, 2000]
    off = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    tok = torch.randint(-3, v + 3, (sum(lens),), generator=g)
    gen = torch.randint(0, 40, (sum(lens),), generator=g)
    add_prompt(h, tok.cuda(), off.cuda())
    add_generated(h, gen.cuda(), off.cuda())
    for _ in range(3):
        add_generated(h, torch.tensor([0, 1, v - 1, -1, v], device="cuda"))
    want = torch.zeros(rows, v, dtype=torch.long)
    for r in range(rows):
        mine = slice(int(off[r]), int(off[r + 1]))
        want[r] += torch.bincount(gen[mine], minlength=v)
        t = tok[mine]
        want[r, t[(t >= 0) & (t < v)].unique()] -= 32768
    want[0, 0] += 3
    want[1, 1] += 3
    want[2, v - 1] += 3
    assert torch.equal(h.cpu().long(), want)
    h[0, 0] = 32766
    h[1, 7] = -2                              # prompt bit and a count of 32766
    for _ in range(3):
        add_generated(h, torch.tensor([0, 7, -1, -1, -1], device="cuda"))
    assert int(h[0, 0]) == 32767 and int(h[1, 7]) == -1 and int(h[0, 1]) == int(want[0, 1])


def test_refusals(cuda_lib):
    from nova_b200.logits import LogitBias, add_generated, adjust_logits, new_history

    x = torch.zeros(2, 100, dtype=torch.float16, device="cuda")
    h = new_history(2, 100)
    one = torch.ones(2, device="cuda")
    m = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    bad = [
        lambda: adjust_logits(x.cpu()),
        lambda: adjust_logits(x.to(torch.bfloat16)),
        lambda: adjust_logits(x[0]),
        lambda: adjust_logits(x, history=h[:, :50]),
        lambda: adjust_logits(x, history=h.int()),
        lambda: adjust_logits(x, repetition=one),
        lambda: adjust_logits(x, history=h, repetition=one.half()),
        lambda: adjust_logits(x, history=h, frequency=one[:1]),
        lambda: adjust_logits(x, allowed=m[:, :3]),
        lambda: adjust_logits(x, allowed=m[:1]),
        lambda: adjust_logits(x, allowed=m[:1].expand(2, 4)),
        lambda: adjust_logits(x, allowed=m, allowed_row=one.long()),
        lambda: adjust_logits(x, allowed_row=one.int()),
        lambda: adjust_logits(x, out=x.float()),
        lambda: adjust_logits(x, bias=LogitBias([{}], 100)),
        lambda: LogitBias([{100: 1.0}, {}], 100),
        lambda: LogitBias([{-1: 1.0}, {}], 100),
        lambda: add_generated(h, torch.zeros(3, dtype=torch.int64, device="cuda")),
        lambda: add_generated(h, torch.zeros(2, dtype=torch.int32, device="cuda")),
        lambda: add_generated(h, torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")

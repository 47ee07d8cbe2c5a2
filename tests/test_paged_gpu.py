"""GPU: the paged int8 cache -- append, read-back and attention -- against plain
64-bit forms, with error bounds derived in paged_reference.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as ref
from oracle import kvquant as okv

pytestmark = pytest.mark.gpu

PAGE, D = 64, 128


def close(got, want, bound, what):
    d = (got.double().cpu() - want).abs()
    worst = (d - bound).max() if d.numel() else torch.tensor(0.0)
    assert torch.isfinite(got).all(), what
    assert worst <= 0, f"{what}: {(d > bound).sum()} of {d.numel()} beyond the bound, by {worst:.3e} (max {d.max():.3e})"


def run_attention(s, window=0, scale=None, windows=None, q=None):
    from nova_b200.paged import paged_attention

    plan = s.plan(windows=windows or (window,))
    lse = torch.empty(s.q.shape[:2], dtype=torch.float32, device="cuda")
    out = paged_attention(s.q.cuda() if q is None else q, s.codes.cuda(), s.scales.cuda(), s.tails.cuda(), plan,
                          window=window, scale=scale, lse_out=lse)
    plan.check_errors()
    return out, lse


ATTENTION = [
    # q_lens, kv_lens, kv_heads, q_heads, window
    ([1], [1], 1, 1, 0),
    ([1], [64], 2, 8, 0),
    ([1], [65], 2, 8, 0),
    ([1, 1, 1, 1], [63, 128, 700, 2049], 2, 8, 0),
    ([1, 1], [5000, 300], 1, 8, 0),
    ([1, 1, 0, 1], [130, 64, 70, 1], 2, 32, 0),
    ([1], [1000], 2, 6, 0),
    ([1, 1], [900, 40], 2, 4, 100),
    ([1], [900], 1, 4, 1),
    ([3, 1], [200, 7], 2, 8, 0),
    ([7, 2, 5], [7, 66, 400], 1, 3, 0),
    ([4], [130], 2, 8, 65),
    ([40, 1, 64], [40, 500, 64], 2, 8, 0),
    ([100, 129], [300, 129], 1, 5, 0),
    ([70], [500], 1, 16, 33),
    ([200, 1, 1], [777, 1000, 64], 2, 8, 0),
    ([300], [300], 2, 2, 0),
    ([257, 130], [1030, 2000], 1, 8, 256),
]


@pytest.mark.parametrize("q_lens,kv_lens,hkv,hq,window", ATTENTION)
def test_attention(cuda_lib, q_lens, kv_lens, hkv, hq, window):
    s = ref.State(q_lens, kv_lens, hkv, hq, seed=len(q_lens) + sum(kv_lens))
    out, lse = run_attention(s, window)
    want, bound, want_lse, lse_bound = ref.attention(s, window)
    close(out, want, bound, "out")
    close(lse, want_lse, lse_bound, "lse")


def test_attention_repeats_bit_for_bit(cuda_lib):
    """Splits are joined in a fixed order, and the workspace is left ready for the next launch."""
    from nova_b200.paged import paged_attention

    s = ref.State([1, 200, 1, 3], [3000, 1500, 700, 4000], 2, 8, seed=5)
    plan, q = s.plan(), s.q.cuda()
    cache = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())
    first = paged_attention(q, *cache, plan)
    for _ in range(5):
        assert torch.equal(first, paged_attention(q, *cache, plan))


def test_attention_strides_scale_and_stream(cuda_lib):
    """Padded and head-major q and out, another scale, a stream of its own."""
    from nova_b200.paged import paged_attention

    s = ref.State([1, 90], [700, 150], 2, 8, seed=9)
    want, bound, _, _ = ref.attention(s, scale=0.05)
    cache = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())
    wide = torch.zeros(91, 3, 8, D, dtype=torch.float16, device="cuda")
    wide[:, 1] = s.q.cuda()
    heads = torch.full((8, 91, D), 7.0, dtype=torch.float16, device="cuda")
    plan = s.plan()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = paged_attention(wide[:, 1], *cache, plan, scale=0.05, out=heads.transpose(0, 1))
    side.synchronize()
    close(out, want, bound, "strided")
    assert out.data_ptr() == heads.data_ptr()


def test_attention_ignores_what_no_query_sees(cuda_lib):
    """Tail slots past the length, other tail buffers and unused pages may hold anything."""
    s = ref.State([1, 150], [200, 150], 2, 8, seed=11)
    want, bound, _, _ = ref.attention(s)
    for i, n in enumerate(s.kv_lens):
        s.tails[s.tail_out[i], :, :, n % PAGE:] = float("nan")
        s.tails[s.tail_out[i] ^ 1] = float("inf")
    used = {p for pages in s.pages for p in pages}
    for p in set(range(s.codes.shape[0])) - used:
        s.scales[p] = float("nan")
    out, _ = run_attention(s)
    close(out, want, bound, "out")


def test_attention_windows_of_one_plan(cuda_lib):
    s = ref.State([1, 64], [600, 400], 2, 8, seed=12)
    for w in (0, 128, 37):
        out, _ = run_attention(s, w, windows=(0, 128, 37))
        want, bound, _, _ = ref.attention(s, w)
        close(out, want, bound, f"window {w}")


def test_attention_in_a_cuda_graph(cuda_lib):
    from nova_b200.paged import paged_attention

    s = ref.State([1, 80, 1], [1500, 500, 3], 2, 8, seed=13)
    want, bound, _, _ = ref.attention(s)
    plan, q = s.plan(), s.q.cuda()
    cache = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())
    out = torch.zeros_like(q)
    paged_attention(q, *cache, plan, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_attention(q, *cache, plan, out=out)
    out.zero_()
    graph.replay()
    close(out, want, bound, "graph")


def append_inputs(s, seed=1, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    t = sum(s.q_lens)
    qkv = (torch.randn(t, (s.hq + 2 * s.hkv) * D, generator=g) * scale).half()
    wq, wk = ((1.0 + 0.2 * torch.randn(D, generator=g)).half() for _ in range(2))
    ang = torch.arange(max(s.kv_lens))[:, None] * 1e4 ** (-torch.arange(0, D, 2) / D)[None]
    ang = torch.cat([ang, ang], 1)
    return qkv, wq, wk, ang.cos().half(), ang.sin().half()


APPEND = [
    # q_lens, kv_lens, kv_heads, q_heads
    ([1], [1], 1, 1),
    ([1], [64], 2, 8),
    ([1, 1, 1], [65, 128, 300], 2, 8),
    ([63], [64], 1, 3),
    ([64, 0, 128], [64, 70, 200], 2, 2),
    ([200, 1, 3], [333, 40, 65], 2, 16),
    ([5, 130], [5, 131], 4, 4),
]


@pytest.mark.parametrize("q_lens,kv_lens,hkv,hq", APPEND)
@pytest.mark.parametrize("plain", [True, False])
def test_append_and_read(cuda_lib, q_lens, kv_lens, hkv, hq, plain):
    """plain: no norm and no rotation, so K and V are the input's own fp16 values
    and codes, scales and tails have to be the framework quantizer's bits."""
    from nova_b200.paged import paged_read, qkv_append

    s = ref.State(q_lens, kv_lens, hkv, hq, seed=3)
    qkv, wq, wk, cos, sin = append_inputs(s)
    if plain:
        wq = wk = cos = sin = None
    t = sum(q_lens)
    x = qkv.view(t, hq + 2 * hkv, D)
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(q_lens, kv_lens)])
    rows = (None, None) if cos is None else (cos[pos], sin[pos])
    want_q, size_q = ref.norm_rope(x[:, :hq], wq, *rows, 1e-6)
    want_k, size_k = ref.norm_rope(x[:, hq:hq + hkv], wk, *rows, 1e-6)
    plan = s.plan()
    codes, scales, tails = s.codes.cuda(), s.scales.cuda(), s.tails.cuda()
    dev = lambda v: None if v is None else v.cuda()  # noqa: E731
    padded = torch.full((t, qkv.shape[1] + 8), float("nan"), dtype=torch.float16, device="cuda")
    padded[:, :qkv.shape[1]] = qkv.cuda()
    before = [v.clone() for v in (codes, scales, tails)]
    for _ in range(2):          # the second run finds the same step: nothing may change
        q = qkv_append(padded[:, :qkv.shape[1]], codes, scales, tails, plan, q_norm_weight=dev(wq), k_norm_weight=dev(wk),
                       cos=dev(cos), sin=dev(sin))
    # fp32 arithmetic (a few 2^-22 of the terms), one rounding to fp16
    close(q, want_q, 2.0 ** -11 * want_q.abs() + 2.0 ** -25 + 2.0 ** -21 * size_q, "q")
    k16 = want_k.half().numpy()
    v16 = x[:, hq + hkv:].numpy()
    off = 2.0 ** -11 * want_k.abs() + 2.0 ** -25 + 2.0 ** -21 * size_k
    touched_pages, touched_tails, t0, row = set(), set(), 0, 0
    k_read, v_read = paged_read(codes, scales, tails, plan)
    codes_c, scales_c, tails_c = codes.cpu(), scales.cpu(), tails.cpu()
    for i, (m, n) in enumerate(zip(q_lens, kv_lens)):
        first = n - m
        for blk in range(first // PAGE, -(-n // PAGE)):
            b0, b1 = blk * PAGE, min(n, blk * PAGE + PAGE)
            old = max(0, min(first, b1) - b0)
            for j, new in ((0, k16), (1, v16)):
                tok = np.concatenate([s.tails[s.tail_in[i], :, j, :old].numpy(),
                                      new[t0 + b0 + old - first:t0 + b1 - first].transpose(1, 0, 2)], axis=1)
                exact = plain or j == 1
                got = (k_read, v_read)[j][row:row + b1 - b0].cpu().numpy().transpose(1, 0, 2)
                if b1 - b0 == PAGE:
                    page = s.pages[i][blk]
                    touched_pages.add(page)
                    qc, mn, st = okv.quantize_int8_token(tok, 64)
                    if exact:
                        assert np.array_equal(codes_c[page, :, j].numpy(), qc)
                        assert np.array_equal(scales_c[page, :, 2 * j].numpy(), mn[:, 0])
                        assert np.array_equal(scales_c[page, :, 2 * j + 1].numpy(), st[:, 0])
                        held = okv.dequantize_int8_token(qc, mn, st, 64)
                        # one rounding against the oracle's two
                        ulp = np.abs(held).astype(np.float64) * 2.0 ** -10 + 2.0 ** -24
                        assert (np.abs(got.astype(np.float64) - held.astype(np.float64)) <= ulp).all()
                    else:   # K may differ by a rounding of fp16 before it is quantized
                        step = st.astype(np.float64)
                        fuzz = off[max(t0, t0 + b0 - first):t0 + b1 - first].amax().item()
                        d = np.abs(got.astype(np.float64) - tok.astype(np.float64))
                        lim = 0.5 * step + 255 * step * 2.0 ** -11 + 4 * fuzz + 2.0 ** -10 * np.abs(tok).astype(np.float64)
                        assert (d <= lim).all(), (d - lim).max()
                else:
                    touched_tails.add(s.tail_out[i])
                    held = tails_c[s.tail_out[i], :, j, :b1 - b0].numpy()
                    assert np.array_equal(held, got)
                    if exact:
                        assert np.array_equal(held, tok)
                    elif m:
                        lim = off[t0 + b0 + old - first:t0 + b1 - first].numpy().transpose(1, 0, 2)
                        d = np.abs(held[:, old:].astype(np.float64)
                                   - want_k[t0 + b0 + old - first:t0 + b1 - first].numpy().transpose(1, 0, 2))
                        assert (d <= lim).all()
                        assert np.array_equal(held[:, :old], tok[:, :old])
            row += b1 - b0
        t0 += m
    assert row == plan.read_rows
    for p in range(codes.shape[0]):          # nothing else was written
        if p not in touched_pages:
            assert torch.equal(codes[p], before[0][p]) and torch.equal(scales[p], before[1][p])
    for b in range(tails.shape[0]):
        if b not in touched_tails:
            assert torch.equal(tails[b], before[2][b])


def test_append_matches_the_quantizer_kernel(cuda_lib):
    """A page holds the bits of quantize_int8 on its 64 tokens (the framework's other int8 cache)."""
    from nova_b200.kvquant import quantize_int8
    from nova_b200.paged import qkv_append

    s = ref.State([192], [192], 2, 2, seed=4)
    qkv, *_ = append_inputs(s)
    x = qkv.cuda()
    x[:, 5] *= 65.0                          # a loud channel
    x[:, 2 * D + 7] = 0.25                   # a constant key channel: step at its floor
    plan = s.plan()
    codes, scales, tails = s.codes.cuda(), s.scales.cuda(), s.tails.cuda()
    qkv_append(x, codes, scales, tails, plan)
    for j in (0, 1):
        t = x.view(192, 6, D)[:, 2 + 2 * j:4 + 2 * j].transpose(0, 1).contiguous()
        qc, mn, st = quantize_int8(t, 64, "token")
        assert torch.equal(codes[s.pages[0], :, j].transpose(0, 1).reshape(2, 192, D), qc)
        assert torch.equal(scales[s.pages[0], :, 2 * j].transpose(0, 1), mn)
        assert torch.equal(scales[s.pages[0], :, 2 * j + 1].transpose(0, 1), st)


def test_cache_token_by_token_equals_chunks(cuda_lib):
    """The same tokens in any pieces leave the same bytes and the same attention of the last token."""
    from nova_b200.paged import PagedKVCache

    hkv, hq, n = 2, 8, 197
    g = torch.Generator().manual_seed(6)
    x = torch.randn(n, (hq + 2 * hkv) * D, generator=g).half().cuda()
    w = (1 + 0.1 * torch.randn(D, generator=g)).half().cuda()
    results = []
    for pieces in ([n], [1] * n, [64, 64, 64, 5], [100, 1, 90, 6], [197 - 1, 1]):
        c = PagedKVCache(2, hkv, hq, num_pages=16, max_requests=3, device="cuda")
        c.add()
        r, at, last = c.add(), 0, None
        for m in pieces:
            plan = c.plan([r], [m])
            q = c.append(1, x[at:at + m], plan, q_norm_weight=w, k_norm_weight=w)
            last = c.attend(1, q, plan)[-1]
            at += m
        plan = c.plan([r], [0], read_from=[0])
        results.append((*c.read(1, plan), last))
        assert not c.codes[0].any()
    for k, v, last in results[1:]:
        assert torch.equal(k, results[0][0]) and torch.equal(v, results[0][1])
        # the last query's row is the same sum in another order of splits
        assert torch.allclose(last.float(), results[0][2].float(), rtol=2.0 ** -9, atol=2.0 ** -12)


def test_refusals(cuda_lib):
    from nova_b200.paged import paged_attention, paged_read, qkv_append

    s = ref.State([1, 2], [70, 130], 2, 8, seed=7)
    plan = s.plan()
    c = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())
    q = s.q.cuda()
    x = torch.zeros(3, 12 * D, dtype=torch.float16, device="cuda")
    bad = [
        lambda: paged_attention(q.float(), *c, plan),
        lambda: paged_attention(q[:2], *c, plan),
        lambda: paged_attention(q.cpu(), *c, plan),
        lambda: paged_attention(q, c[0][:, :1].contiguous(), *c[1:], plan),
        lambda: paged_attention(q, c[0][:1], c[1][:1], c[2], plan),          # fewer pages than the plan uses
        lambda: paged_attention(q, c[0], c[1], c[2][:1], plan),
        lambda: paged_attention(q, c[0], c[1].float(), c[2], plan),
        lambda: paged_attention(q, c[0].cpu(), c[1].cpu(), c[2].cpu(), plan),
        lambda: paged_attention(q, *c, plan, window=5),
        lambda: paged_attention(q, *c, plan, scale=0.0),
        lambda: paged_attention(q, *c, plan, out=torch.empty(3, 8, D, device="cuda")),
        lambda: paged_attention(q, *c, plan, lse_out=torch.empty(3, 8, device="cuda", dtype=torch.float16)),
        lambda: paged_attention(torch.zeros(3, 8, D + 1, dtype=torch.float16, device="cuda")[..., :D], *c, plan),
        lambda: qkv_append(x[:, :-1], *c, plan),
        lambda: qkv_append(x.float(), *c, plan),
        lambda: qkv_append(x, *c, plan, cos=x),
        lambda: qkv_append(x, *c, plan, q_norm_weight=x[0, :64]),
        lambda: qkv_append(x, *c, plan, cos=x[:1, :D].contiguous(), sin=x[:1, :D].contiguous()),   # table too short
        lambda: paged_read(c[0], c[1][:1], c[2], plan),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")


def test_empty_step(cuda_lib):
    from nova_b200.paged import paged_attention, paged_read, qkv_append

    s = ref.State([0, 0], [64, 0], 1, 4, seed=8)
    plan = s.plan()
    c = (s.codes.cuda(), s.scales.cuda(), s.tails.cuda())
    q = qkv_append(torch.zeros(0, 6 * D, dtype=torch.float16, device="cuda"), *c, plan)
    assert q.shape == (0, 4, D) and paged_attention(q, *c, plan).shape == (0, 4, D)
    k, v = paged_read(*c, plan)
    assert k.shape == v.shape == (0, 1, D)

"""GPU: the request server -- paged cache, adapters and logit controls run
together -- against a plain 64-bit decoder on the dequantized weights that
quantizes the same pages."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kvquant as okv

pytestmark = pytest.mark.gpu

PAGE = 64


def small_cfg():
    from nova_b200.decoder import DecoderConfig

    return DecoderConfig(vocab_size=4096, hidden_size=512, num_hidden_layers=2, num_attention_heads=8,
                         num_key_value_heads=2, head_dim=128, intermediate_size=1024)


class PlainDecoder:
    """One request, token pieces at a time, 64 bits, K and V of full pages replaced by their int8 values."""

    def __init__(self, weights, bank=None, adapter=-1):
        from nova_b200.decoder import deinterleave_gate_up, rope_tables
        from nova_b200.kernels import build_nf4_lut
        from nova_b200.quant import dequantize_nf4, nf4_codebook

        self.cfg, lut = weights.cfg, build_nf4_lut(nf4_codebook()).cuda()
        deq = lambda p, a: dequantize_nf4(p.contiguous(), a.contiguous(), lut).double().cpu()  # noqa: E731
        self.layers = []
        for li, w in enumerate(weights.layers):
            gp, ga, up, ua = deinterleave_gate_up(w.gate_up.packed, w.gate_up.absmax)
            qkv, o = deq(w.qkv.packed, w.qkv.absmax), deq(w.o.packed, w.o.absmax)
            if adapter >= 0:
                r, s = bank.ranks[adapter], float(bank.scaling[adapter])
                qkv = qkv + s * bank.qkv_b[li][adapter, :, :r].double().cpu() @ bank.qkv_a[li][adapter, :r].double().cpu()
                o = o + s * bank.o_b[li][adapter, :, :r].double().cpu() @ bank.o_a[li][adapter, :r].double().cpu()
            self.layers.append(dict(qkv=qkv, o=o, gate=deq(gp, ga), up=deq(up, ua), down=deq(w.down.packed, w.down.absmax),
                                    **{n: getattr(w, n).double().cpu() for n in ("input_ln", "post_ln", "q_norm", "k_norm")}))
        self.embed, self.head = weights.embed.double().cpu(), deq(weights.lm_head.packed, weights.lm_head.absmax)
        self.norm = weights.final_norm.double().cpu()
        self.cos, self.sin = (t.double().cpu() for t in rope_tables(2048, 128, self.cfg.rope_theta, "cpu"))
        self.kv = [[torch.zeros(0, 2, 128, dtype=torch.float64) for _ in range(2)] for _ in self.layers]

    def _rms(self, x, w):
        return x / (x.pow(2).mean(-1, keepdim=True) + self.cfg.rms_norm_eps).sqrt() * w

    def _rope(self, x, pos):
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        return x * c + torch.cat([-x[..., 64:], x[..., :64]], -1) * s

    def advance(self, tokens):
        cfg, x = self.cfg, self.embed[torch.tensor(tokens)]
        n0 = self.kv[0][0].shape[0]
        pos = torch.arange(n0, n0 + len(tokens))
        for li, w in enumerate(self.layers):
            h = (self._rms(x, w["input_ln"]) @ w["qkv"].t()).view(len(tokens), -1, 128)
            hq, hk = cfg.num_attention_heads, cfg.num_key_value_heads
            q = self._rope(self._rms(h[:, :hq], w["q_norm"]), pos)
            k = self._rope(self._rms(h[:, hq:hq + hk], w["k_norm"]), pos)
            self.kv[li][0] = torch.cat([self.kv[li][0], k.half().double()])
            self.kv[li][1] = torch.cat([self.kv[li][1], h[:, hq + hk:].half().double()])
            vals = []
            for t in self.kv[li]:
                full = t.shape[0] // PAGE * PAGE
                a = t[:full].transpose(0, 1).half().numpy()
                back = okv.dequantize_int8_token(*okv.quantize_int8_token(a, 64), 64) if full else a
                vals.append(torch.cat([torch.from_numpy(np.asarray(back)).double().transpose(0, 1), t[full:]]))
            g = hq // hk
            kk, vv = (v.repeat_interleave(g, 1) for v in vals)
            s = torch.einsum("qhd,khd->hqk", q, kk) / 128 ** 0.5
            s = s.masked_fill(torch.arange(kk.shape[0])[None] > pos[:, None], -float("inf"))
            o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), vv).reshape(len(tokens), -1)
            x = x + o @ w["o"].t()
            h = self._rms(x, w["post_ln"])
            a = h @ w["gate"].t()
            x = x + (a * torch.sigmoid(a) * (h @ w["up"].t())) @ w["down"].t()
        return self._rms(x[-1:], self.norm) @ self.head.t()


def test_requests_match_a_plain_decoder(cuda_lib):
    """Three requests of different lengths and adapters, prompt chunks mixed with decoding.  The server's
    activations are fp16: logits within 2 % of their range (the graph decoder's criterion is of that kind)."""
    from nova_b200.decoder import DecoderWeights
    from nova_b200.serving import AdapterBank, RequestServer

    cfg = small_cfg()
    W = DecoderWeights.random_init(cfg, seed=3, norm_jitter=0.1)
    bank = AdapterBank.random_init(cfg, [8, 13], seed=4, std=0.1)
    srv = RequestServer(W, num_pages=64, max_requests=4, adapters=bank, chunk=100)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (130, 1, 263)]
    adapters = [1, -1, 0]
    rids = [srv.submit(p, adapter=a) for p, a in zip(prompts, adapters)]
    plain = {r: PlainDecoder(W, bank, a) for r, a in zip(rids, adapters)}
    todo = {r: list(p) for r, p in zip(rids, prompts)}
    last, seen = {}, []
    for _ in range(6):
        pieces = {r: [todo[r].pop(0) for _ in range(min(100, len(todo[r])))] or [last[r]] for r in rids}
        got = srv.step()
        for i, r in enumerate([r for r in rids if not todo[r]]):
            want = plain[r].advance(pieces[r])[0]
            lg = srv.raw_logits[i].double().cpu()
            seen.append(r)
            assert (lg - want).abs().max() <= 0.02 * want.abs().max(), (r, float((lg - want).abs().max()))
            assert got[r] == int(srv.logits[i].argmax())
            last[r] = got[r]
        for r in rids:
            if todo[r]:
                plain[r].advance(pieces[r])
        assert set(got) == {r for r in rids if not todo[r]}
    assert set(seen) == set(rids)
    assert [srv.length(r) for r in rids] == [130 + 4, 1 + 5, 263 + 3]


def test_controls_and_release(cuda_lib):
    from nova_b200.decoder import DecoderWeights
    from nova_b200.serving import RequestServer

    cfg = small_cfg()
    W = DecoderWeights.random_init(cfg, seed=6)
    srv = RequestServer(W, num_pages=8, max_requests=2)
    words = -(-cfg.vocab_size // 32)
    only = torch.zeros(words, dtype=torch.int32, device="cuda")
    only[3] = 1 << 5                                            # token 101 alone
    a = srv.submit([1, 2, 3], allowed=only)
    b = srv.submit([5] * 70, bias={7: 1e4})
    got = srv.step()
    assert got == {a: 101, b: 7}
    srv.set_allowed(a, None)
    srv.step()
    for _ in range(3):
        got = srv.step([b])
        assert set(got) == {b} and got[b] == 7                  # counted each time, penalties are off
    slot = srv._requests[b].slot
    assert int(srv.history[slot, 7]) == 5 and int(srv.history[slot, 5]) == -32768
    with pytest.raises(RuntimeError):
        srv.submit([1])
    free = srv.cache.free_pages()
    srv.release(b)
    assert srv.cache.free_pages() == free + 1
    c = srv.submit([9], frequency=1e4, repetition=2.0)          # the slot's old history is gone
    first = srv.step([c])[c]
    assert srv.step([c])[c] != first
    with pytest.raises(ValueError):
        srv.submit([])
    with pytest.raises(ValueError):
        srv.submit([1], adapter=0)
    srv.release(c)
    d = srv.submit([1] * 2000)                                  # 8 pages hold its first chunk only
    assert srv.step([d]) == {}
    with pytest.raises(RuntimeError, match="pages"):
        srv.step([d])
    assert srv.length(d) == 512 and len(srv._requests[d].todo) == 2000 - 512


def test_sampling_is_reproducible(cuda_lib):
    from nova_b200.decoder import DecoderWeights
    from nova_b200.serving import RequestServer

    W = DecoderWeights.random_init(small_cfg(), seed=6)
    runs = []
    for _ in range(2):
        srv = RequestServer(W, num_pages=8, max_requests=2, temperature=0.8, top_k=20, top_p=0.9, seed=11)
        r = [srv.submit([1, 2, 3]), srv.submit([4] * 80)]
        runs.append([[got[i] for i in r] for got in (srv.step() for _ in range(6))])
    assert runs[0] == runs[1]

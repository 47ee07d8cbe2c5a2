"""GPU: the request server when a step fails on the host or a kernel reports an
error.  Nothing here makes a GPU fail: exceptions are raised and error words set
by the test."""

from __future__ import annotations

import pytest
import torch

from test_serving_gpu import small_cfg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights(cuda_lib):
    from nova_b200.decoder import DecoderWeights

    return DecoderWeights.random_init(small_cfg(), seed=6)


def server(weights, **kw):
    from nova_b200.serving import RequestServer

    srv = RequestServer(weights, num_pages=32, max_requests=3, chunk=100, **kw)
    g = torch.Generator().manual_seed(1)
    for n, controls in ((250, {"repetition": 1.3}), (63, {"frequency": 0.7, "presence": 0.2}), (1, {"bias": {7: 2.0}})):
        srv.submit(torch.randint(0, 4096, (n,), generator=g).tolist(), **controls)
    return srv


def state(srv):
    return ({i: (srv.length(i), list(r.todo)) for i, r in srv._requests.items()}, srv.cache.free_pages(),
            srv.history.cpu().clone(), srv.tokens.cpu().clone())


def same(x, y):
    return x[:2] == y[:2] and torch.equal(x[2], y[2]) and torch.equal(x[3], y[3])


def fail_at(srv, monkeypatch, layer):
    """Every attention from `layer` on raises, once."""
    attend = srv.cache.attend

    def broken(li, *a, **kw):
        if li == layer:
            monkeypatch.setattr(srv.cache, "attend", attend)
            raise MemoryError("no memory for this layer")
        return attend(li, *a, **kw)

    monkeypatch.setattr(srv.cache, "attend", broken)


def test_a_step_that_raises_can_be_taken_again(weights, monkeypatch):
    """Failures in the middle of prompt chunks, of the steps in which pages fill, and of decoding: every request is
    as it was, and the steps that follow give the bits of a server that never failed."""
    good, bad = server(weights), server(weights)
    for i in range(7):
        before = state(bad)
        fail_at(bad, monkeypatch, i % 2)
        with pytest.raises(MemoryError):
            bad.step()
        assert same(state(bad), before)
        want = good.step()
        assert bad.step() == want
        if want:
            assert torch.equal(good.raw_logits, bad.raw_logits) and torch.equal(good.logits, bad.logits)
    assert same(state(good), state(bad))


@pytest.mark.parametrize("kernel", ["attention", "gemm"])
def test_error_words_are_read(weights, monkeypatch, kernel):
    """What a bounded wait that gives up leaves in a workspace stops the step, prompt chunks without a token included."""
    good, bad = server(weights), server(weights)
    attend = bad.cache.attend
    for i in range(4):
        before = state(bad)
        requests = list(bad._requests)[:1] if i == 0 else None      # first a chunk of the longest prompt alone

        def reports(li, q, plan, **kw):
            out = attend(li, q, plan, **kw)
            if li == 1:
                (plan.workspace[:4] if kernel == "attention" else bad.gemm_ws[4:8]).view(torch.int32).fill_(2)
            return out

        monkeypatch.setattr(bad.cache, "attend", reports)
        with pytest.raises(RuntimeError, match="bounded wait"):
            bad.step(requests)
        monkeypatch.setattr(bad.cache, "attend", attend)
        assert same(state(bad), before)
        assert bad.step(requests) == good.step(requests)
    assert same(state(good), state(bad))


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_mask_that_leaves_nothing_gives_no_token(weights, temperature):
    """An empty mask, a mask of which a bias takes the last token: no forbidden token comes out, nobody loses one, and
    the others go on once the request has another mask or is left out."""
    cfg = small_cfg()
    srv = server(weights, temperature=temperature)
    words = -(-cfg.vocab_size // 32)
    a, b, c = srv._requests
    srv.step()
    srv.step()
    empty, one = (torch.zeros(words, dtype=torch.int32, device="cuda") for _ in range(2))
    one[3] = 1 << 5                                           # token 101 alone
    srv.set_allowed(b, empty)
    before = state(srv)
    with pytest.raises(RuntimeError, match=rf"no token is left for requests \[{b}\]"):
        srv.step()
    assert same(state(srv), before)
    assert set(srv.step([a, c])) == {a, c}
    srv.set_allowed(b, one)
    assert srv.step()[b] == 101
    srv.biases[srv._requests[b].slot] = {101: -float("inf")}
    before = state(srv)
    with pytest.raises(RuntimeError, match="no token is left"):
        srv.step([b])
    assert same(state(srv), before)


def test_both_error_words_are_cleared(weights):
    good, bad = server(weights), server(weights)
    bad.gemm_ws[4:8].view(torch.int32).fill_(3)
    plan = bad.cache.plan
    bad.cache.plan = lambda *a, **kw: (bad.cache.__dict__.pop("plan"), set_word(plan(*a, **kw)))[1]
    with pytest.raises(RuntimeError, match="bounded wait"):
        bad.step()
    assert bad.step() == good.step() and same(state(good), state(bad))


def set_word(plan):
    plan.workspace[:4].view(torch.int32).fill_(2)
    return plan

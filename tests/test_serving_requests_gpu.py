"""GPU: what the request server refuses, and which requests it names when a step
cannot be taken."""

from __future__ import annotations

import pytest
import torch

from test_serving_gpu import small_cfg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights(cuda_lib):
    from nova_b200.decoder import DecoderWeights

    return DecoderWeights.random_init(small_cfg(), seed=6)


def test_a_refused_request_leaves_nothing(weights):
    from nova_b200.serving import RequestServer

    srv = RequestServer(weights, num_pages=8, max_requests=1, max_len=100)
    nan = float("nan")
    for prompt, kw in (([1] * 101, {}), ([1], {"repetition": nan}), ([1], {"repetition": 0}), ([1], {"frequency": "much"}),
                       ([1], {"bias": {7: "more"}}), ([1], {"bias": {-1: 1.0}}), ([1], {"adapter": 0}),
                       ([1], {"allowed": [1, 2]}), ([4096], {}), (["one"], {})):
        with pytest.raises(ValueError):
            srv.submit(prompt, **kw)
        assert not srv._requests and not srv.cache._requests
    a = srv.submit([1] * 100)                                  # the one slot is still free
    assert set(srv.step()) == {a} and srv.length(a) == 100


def test_steps_name_the_requests_that_stop_them(weights):
    from nova_b200.serving import RequestError, RequestServer

    srv = RequestServer(weights, num_pages=4, max_requests=4, max_len=130, chunk=128)
    a, b, c = srv.submit([1] * 128), srv.submit([2] * 127), srv.submit([3])
    with pytest.raises(RequestError, match="pages") as e:
        srv.submit([4] * 64)                                   # 128 + 127 + 64 tokens fill 2, 1 and 1 pages: one to go
        d = max(srv._requests)
        srv.step()
        srv.step()
    assert e.value.requests == [b]
    srv.release(d)
    got = srv.step()
    assert set(got) == {a, b, c}
    srv.step()
    with pytest.raises(RequestError, match="max_len 130") as e:
        srv.step()
    assert e.value.requests == [a] and srv.length(a) == 130 and srv.length(b) == 129
    assert set(srv.step([b, c])) == {b, c}
    srv.release(a)
    with pytest.raises(RequestError) as e:
        srv.step()
    assert e.value.requests == [b]


def test_more_than_one_request_without_a_token(weights):
    from nova_b200.serving import RequestError, RequestServer

    cfg = small_cfg()
    srv = RequestServer(weights, num_pages=4, max_requests=3)
    none = torch.zeros(-(-cfg.vocab_size // 32), dtype=torch.int32, device="cuda")
    a, b, c = srv.submit([1], allowed=none), srv.submit([2]), srv.submit([3], allowed=none)
    with pytest.raises(RequestError) as e:
        srv.step()
    assert e.value.requests == [a, c] and set(srv.step([b])) == {b}

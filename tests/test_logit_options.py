"""Options that change logits before a token is chosen: what they refuse, how masks are packed, how a request that no token may
continue ends.  No GPU."""

import math

import numpy as np
import pytest

from inf_engine_b200.sampling import SamplingConfig, allowed_words


def test_defaults_ask_for_nothing():
    c = SamplingConfig()
    c.validate()
    assert not (c.adjusts or c.keeps_history or c.windowed)
    assert SamplingConfig(repetition_penalty=1.3).windowed and not SamplingConfig(repetition_penalty=1.3).adjusts
    h = SamplingConfig(repetition_penalty=1.3, repetition_scope="history")
    assert h.keeps_history and h.adjusts and not h.windowed
    assert not SamplingConfig(repetition_scope="history").adjusts
    assert SamplingConfig(presence_penalty=-0.5).keeps_history and SamplingConfig(frequency_penalty=0.1).keeps_history
    b = SamplingConfig(logit_bias={3: 1.5})
    assert b.adjusts and not b.keeps_history


@pytest.mark.parametrize("bad", [
    dict(repetition_scope="all"), dict(presence_penalty=math.inf), dict(frequency_penalty=math.nan), dict(repetition_penalty=math.inf),
    dict(repetition_penalty=0.0), dict(logit_bias={3: math.nan}), dict(logit_bias={3: 1e38}), dict(logit_bias={-1: 1.0}),
    dict(logit_bias={"a": 1.0}), dict(logit_bias={True: 1.0})])
def test_refused(bad):
    with pytest.raises(ValueError):
        SamplingConfig(**bad).validate()


def bits(words, v):
    return np.unpackbits(words.view(np.uint8), bitorder="little")[:v].astype(bool)


@pytest.mark.parametrize("v", [1, 31, 32, 33, 100, 1000])
def test_allowed_words(v):
    rng = np.random.default_rng(v)
    mask = rng.random(v) < 0.4
    ids = np.nonzero(mask)[0]
    for form in (mask, ids, list(map(int, ids)), set(map(int, ids)), np.repeat(ids, 2)):
        w = allowed_words(form, v)
        assert w.dtype == np.int32 and w.shape == (-(-v // 32),) and np.array_equal(bits(w, v), mask)
    assert not allowed_words([], v).any()
    for bad in ([v], [-1], np.zeros(v + 1, bool), np.zeros((1, v), bool), [0.5], np.zeros((2, 2), int)):
        with pytest.raises(ValueError):
            allowed_words(bad, v)


def test_a_request_that_no_token_may_continue_ends():
    from inf_engine_b200.cache.manager import CacheManager, CacheRequirement
    from inf_engine_b200.engine.scheduler import Request, Scheduler
    import torch
    cache = CacheManager([CacheRequirement(kind="kv", n_kv_heads=1, head_dim=8, dtype=torch.float32)], 4, 16, 4, 8)
    s = Scheduler(cache, 64)
    a, b = Request(0, [1, 2, 3], 5), Request(1, [4, 5], 5)
    assert s.submit(a) and s.submit(b)
    plan = s.plan()
    for e in plan.entries:
        cache.advance(e.request.req_id, cache.lengths[e.request.req_id] + len(e.tokens))
    done = s.commit(plan, {0: None, 1: 7}, 2.0)
    assert done == [a] and a.error == "no token is allowed" and a.generated == [] and a.finish_time == 2.0
    assert b.generated == [7] and s.running == [b] and 0 not in cache.slots

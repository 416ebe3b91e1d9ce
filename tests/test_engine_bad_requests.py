"""One request that cannot go on ends alone: options refused at submit, functions of allowed tokens that raise.  No GPU: the engine's own
queue, plans and commits run over a runner and a sampler that only count."""

import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from inf_engine_b200.cache.manager import CacheManager, CacheRequirement
from inf_engine_b200.engine.engine import Engine
from inf_engine_b200.engine.scheduler import Request, Scheduler
from inf_engine_b200.sampling import SamplingConfig, pack_rows, uniform_of

VOCAB = 100
BAD = [dict(repetition_penalty=1.3, repetition_scope="all"), dict(mode="temperature", temperature=0.0),
       dict(mode="temperature", temperature=math.nan), dict(temperature="hot", mode="top_k"), dict(mode="top_p", top_p=0.0),
       dict(mode="top_p", top_p=math.nan), dict(mode="top_p", top_p=None), dict(mode="top_k", top_k="many"), dict(mode="top_k", top_k=math.inf), dict(seed=0.5), dict(seed="x"), dict(repetition_penalty=-1.0),
       dict(repetition_penalty="2"), dict(repetition_penalty=1e-300), dict(repetition_penalty=1e39, repetition_scope="history"),
       dict(presence_penalty=1e300), dict(frequency_penalty=-1e31), dict(presence_penalty=None), dict(logit_bias={3: "1"}),
       dict(logit_bias={3: 10 ** 400}), dict(logit_bias={3: None}), dict(logit_bias=[3, 1.0]), dict(logit_bias={VOCAB: 1.0})]


def engine(chosen, sampling=None, **kw):
    """An engine whose model answers ``chosen(request)`` for every row."""
    cache = CacheManager([CacheRequirement(kind="kv", n_kv_heads=1, head_dim=8, dtype=torch.float32)], 4, 64, 8, 16)

    def step(entries):
        for e in entries:
            cache.advance(e.rid, cache.lengths[e.rid] + len(e.tokens))
        return torch.zeros(sum(len(e.want) for e in entries), VOCAB)

    e = Engine.__new__(Engine)
    e.runner = SimpleNamespace(cache=cache, spec=SimpleNamespace(vocab_size=VOCAB, max_positions=64), step=step,
                               graphs=SimpleNamespace(replays=0))
    e.cfg = sampling or SamplingConfig()
    e.scheduler = Scheduler(cache, 64, max_batch=8)
    e.adjuster = SimpleNamespace(history=None)
    e.stats = {"steps": 0, "prefill_tokens": 0, "decode_tokens": 0, "preemptions": 0}
    e.pipeline, e._pending, e._trace, e._nvtx = False, None, None, False
    e.sampler = SimpleNamespace(sample=lambda logits, configs, keys, contexts, adjuster, rows: torch.tensor(
        [chosen(r) for r, _, _, _ in rows] if rows else [0] * len(configs), dtype=torch.int32))
    e.runner.step_and_sample = lambda entries, rows: (step(entries), torch.zeros(len(rows), dtype=torch.int32))
    return e


def test_the_fake_has_the_names_that_steps_use():
    from inf_engine_b200.engine.batch import StepEntry
    assert StepEntry("x", [1], [0]).want == [0]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_options_that_cannot_be_used_are_refused_at_submit(bad):
    c = SamplingConfig(**bad)
    e = engine(lambda r: 7)
    r, other = Request(0, [1, 2], 3, sampling=c), Request(1, [1, 2], 3)
    assert not e.submit(r) and r.error and e.submit(other)
    for _ in range(20):
        if e.has_work:
            e.step()
    assert e.completed == [other] and len(other.generated) == 3
    if bad.get("logit_bias") != {VOCAB: 1.0}:
        with pytest.raises(ValueError):
            c.validate()


def test_an_engines_own_options_are_checked_too():
    with pytest.raises(ValueError, match="vocabulary"):
        Engine(SimpleNamespace(spec=SimpleNamespace(vocab_size=VOCAB)), sampling=SamplingConfig(logit_bias={VOCAB: 1.0}))
    with pytest.raises(ValueError, match="scope"):
        Engine(SimpleNamespace(spec=SimpleNamespace(vocab_size=VOCAB)), sampling=SamplingConfig(repetition_scope="all"))


@pytest.mark.parametrize("good", [dict(seed=np.int64(-5)), dict(seed=1 << 70), dict(seed=-1), dict(top_k=np.int32(4)), dict(top_p=np.float32(0.5)),
                                  dict(logit_bias={np.int64(3): np.float32(2)}), dict(logit_bias={}), dict(repetition_penalty=2), dict(top_p=0.0)], ids=str)
def test_options_of_other_number_types_are_taken(good):
    c = SamplingConfig(mode="top_k", **good)
    c.validate()
    row = pack_rows([c], [9], VOCAB).view(np.uint32)[0]
    assert int(row[3]) | int(row[4]) << 32 == int(c.seed) % (1 << 64) and 0 <= uniform_of(int(c.seed), 9) < 1


def raising(said):
    if len(said) == 2:
        raise RuntimeError("no rule for this")
    return [7]


@pytest.mark.parametrize("allowed,n,why", [
    (raising, 2, "RuntimeError: no rule for this"), (lambda g: [VOCAB], 0, "outside the vocabulary"), (lambda g: 5, 0, "allowed_tokens"),
    (lambda g: np.ones(VOCAB + 1, bool), 0, "truth value"), (lambda g: [7] if len(g) < 3 else [], 3, "no token is allowed"),
    (lambda g: [8], 0, "no allowed token has a logit above -inf")])
def test_a_request_that_cannot_go_on_ends_alone(allowed, n, why):
    e = engine(lambda r: 7)
    good = [Request(i, [1, 2, 3], 6, allowed_tokens=(lambda g: [7]) if i == 2 else None) for i in range(3)]
    bad = Request(9, [4, 5], 6, allowed_tokens=allowed)
    for r in (good[0], bad, *good[1:]):
        assert e.submit(r)
    for _ in range(40):
        if e.has_work:
            e.step(1.0)
    assert not e.has_work and bad in e.completed and bad.generated == [7] * n and why in bad.error and bad.finish_time == 1.0
    assert all(r in e.completed and len(r.generated) == 6 and r.error is None for r in good)
    assert not e.runner.cache.slots


def test_interrupts_are_not_taken_for_the_requests_fault():
    def stop(said):
        raise KeyboardInterrupt
    e = engine(lambda r: 7)
    assert e.submit(Request(0, [1], 2, allowed_tokens=stop))
    with pytest.raises(KeyboardInterrupt):
        e.step()


@pytest.mark.gpu
@pytest.mark.parametrize("pipeline", [True, False])
def test_neighbours_of_bad_requests_are_served(tmp_path, pipeline):
    from helpers import make_model_dir
    e = Engine.from_dir(make_model_dir(tmp_path, "tiny_a"), dtype="float32", n_total_blocks=64, block_size=8, max_requests=4, pipeline=pipeline)
    alone = e.run_offline([Request(0, [5, 6, 7], 8)])[0]
    e.completed.clear()
    bad = [Request(1, [5, 6], 8, sampling=SamplingConfig(repetition_penalty=1.3, repetition_scope="all")),
           Request(2, [5, 6], 8, allowed_tokens=raising), Request(3, [5, 6], 8, allowed_tokens=lambda g: [256])]
    good = Request(0, [5, 6, 7], 8)
    out = e.run_offline([*bad, good])
    assert out[0] == alone and good.error is None
    assert out[1] == [] and "scope" in bad[0].error and out[2] == [7, 7] and "no rule" in bad[1].error
    assert out[3] == [] and "vocabulary" in bad[2].error
    e.completed.clear()
    assert e.run_offline([Request(0, [5, 6, 7], 8)])[0] == alone

"""Generation under penalties over what a request has said, biases and masks, through the engine, against a plain greedy loop over
the plain implementation's logits in 64 bits.  The float32 engine and the plain implementation differ by the order of sums, F32_ABS
of the largest logit; a token may differ from the plain loop's only where two adjusted logits are nearer than twice that, and
the comparison then goes on from the engine's token."""

import pytest
import torch

import plain_llama
from helpers import F32_ABS, make_model_dir, plain_inputs, random_tokens

pytestmark = pytest.mark.gpu


def options(i, vocab):
    from inf_engine_b200 import SamplingConfig
    return [None,
            SamplingConfig(presence_penalty=0.6, frequency_penalty=0.3),
            SamplingConfig(repetition_penalty=1.4, repetition_scope="history"),
            SamplingConfig(logit_bias={5: 3.0, vocab - 1: 2.0, 7: -4.0}),
            SamplingConfig(repetition_penalty=1.2, repetition_scope="history", presence_penalty=-0.2, frequency_penalty=0.5,
                           logit_bias={0: 1.0, 9: 1.0}),
            SamplingConfig(repetition_penalty=1.3, frequency_penalty=0.4)][i % 6]      # windowed, and a history beside it


def adjusted(row, prompt, said, c, allowed):
    """A row of logits as the options leave it (float64)."""
    x = row.double().clone()
    if c is not None:
        if c.repetition_penalty != 1.0:
            for t in set(said[-256:] if c.repetition_scope == "window" else prompt + said):
                x[t] = x[t] * c.repetition_penalty if x[t] < 0 else x[t] / c.repetition_penalty
        for t in set(said):
            x[t] -= c.frequency_penalty * said.count(t) + c.presence_penalty
        for t, v in (c.logit_bias or {}).items():
            x[t] += v
    if allowed is not None:
        keep = torch.full_like(x, -torch.inf)
        keep[list(allowed)] = x[list(allowed)]
        x = keep
    return x


def check(weights, config, requests, out, allowed=None):
    for r in requests:
        logits = plain_llama.forward_logits(weights, config, r.prompt_ids + out[r.req_id])
        slack = 4 * F32_ABS * max(1.0, float(logits.abs().max()))
        for j, t in enumerate(out[r.req_id]):
            said = out[r.req_id][:j]
            x = adjusted(logits[len(r.prompt_ids) + j - 1], r.prompt_ids, said, r.sampling, allowed(r, said) if allowed else None)
            assert float(x.max() - x[t]) <= slack, f"request {r.req_id} token {j}"


@pytest.mark.parametrize("pipeline", [True, False])
@pytest.mark.parametrize("pages", [200, 14])              # enough for all; so few that requests give way and come back
def test_penalties_and_biases(tmp_path, pipeline, pages):
    from inf_engine_b200 import Engine, Request
    d = make_model_dir(tmp_path, "tiny_a")
    config, weights = plain_inputs(d)
    engine = Engine.from_dir(d, dtype="float32", n_total_blocks=pages, block_size=8, max_requests=5, max_tokens_per_step=32,
                             pipeline=pipeline)
    requests = [Request(i, random_tokens(256, 3 + 5 * i, 70 + i), 25, sampling=options(i, 256)) for i in range(9)]
    out = engine.run_offline(requests)
    assert all(len(out[r.req_id]) == 25 for r in requests)
    if pages == 14:
        assert sum(r.preemptions for r in requests) > 0
    check(weights, config, requests, out)
    # a second run through slots that others' histories have been in
    again = [Request(100 + i, r.prompt_ids, 25, sampling=r.sampling) for i, r in enumerate(reversed(requests))]
    out2 = engine.run_offline(again)
    check(weights, config, again, {r.req_id: out2[r.req_id] for r in again})


def test_steps_run_ahead_under_penalties(tmp_path):
    from inf_engine_b200 import Engine, Request
    d = make_model_dir(tmp_path, "tiny_a")
    engine = Engine.from_dir(d, dtype="float32", n_total_blocks=64, block_size=8, max_requests=2)
    engine.submit(Request(0, [1, 2, 3], 12, sampling=options(1, 256)))
    ahead = 0
    while engine.has_work:
        engine.step()
        ahead += engine._pending is not None
    assert ahead >= 10


def test_sampling_modes_see_the_adjusted_logits(tmp_path):
    """All but one token pushed far down: whatever the mode draws is that token; a mask does the same."""
    from inf_engine_b200 import Engine, Request, SamplingConfig
    d = make_model_dir(tmp_path, "tiny_a")
    engine = Engine.from_dir(d, dtype="bfloat16", n_total_blocks=64, block_size=8, max_requests=4)
    bias = {t: -1e6 for t in range(256) if t != 77}
    for mode in ("temperature", "top_k", "top_p", "greedy"):
        c = SamplingConfig(mode=mode, temperature=1.5, logit_bias=bias, seed=3)
        out = engine.run_offline([Request(0, [5, 6], 6, sampling=c),
                                  Request(1, [5, 6], 6, sampling=SamplingConfig(mode=mode, temperature=1.5, seed=4), allowed_tokens=lambda g: [77])])
        assert out[0] == [77] * 6 and out[1] == [77] * 6
        engine.scheduler.completed.clear()


def test_masks(tmp_path):
    from inf_engine_b200 import Engine, Request, SamplingConfig
    d = make_model_dir(tmp_path, "tiny_b")
    config, weights = plain_inputs(d)
    v = config["vocab_size"]
    engine = Engine.from_dir(d, dtype="float32", n_total_blocks=64, block_size=8, max_requests=4)

    def grammar(said):                  # even tokens first, then odd ones, then anything, then nothing
        if len(said) >= 9:
            return []
        return None if 5 <= len(said) < 7 else list(range(len(said) % 2, v, 2))

    requests = [Request(0, [3, 4, 5], 20, allowed_tokens=grammar),
                Request(1, [9, 8], 8),
                Request(2, [7], 8, sampling=SamplingConfig(presence_penalty=0.5), allowed_tokens=lambda g: range(len(g), 40))]
    out = engine.run_offline(requests)
    assert len(out[0]) == 9 and requests[0].error == "no token is allowed" and requests[1].error is None
    assert all(t % 2 == j % 2 for j, t in enumerate(out[0]) if not 5 <= j < 7)
    check(weights, config, requests, out, lambda r, said: r.allowed_tokens(said) if r.allowed_tokens else None)


def test_a_request_submitted_again_has_a_new_history(tmp_path):
    from inf_engine_b200 import Engine, Request, SamplingConfig
    d = make_model_dir(tmp_path, "tiny_a")
    config, weights = plain_inputs(d)
    engine = Engine.from_dir(d, dtype="float32", n_total_blocks=64, block_size=8, max_requests=1)
    r = Request(0, random_tokens(256, 9, 1), 8, sampling=SamplingConfig(repetition_penalty=1.5, repetition_scope="history", frequency_penalty=0.5))
    for seed in (1, 2, 3):
        r.prompt_ids, r.generated, r.start_time, r.finish_time = random_tokens(256, 9, seed), [], 0.0, 0.0
        out = engine.run_offline([r])
        check(weights, config, [r], out)
        engine.scheduler.completed.clear()


def test_requests_admitted_together_keep_their_masks(tmp_path):
    """A mask needs its request's tokens on the host, wherever in the queue it stands when a step admits it."""
    from inf_engine_b200 import Engine, Request
    d = make_model_dir(tmp_path, "tiny_a")
    engine = Engine.from_dir(d, dtype="float32", n_total_blocks=128, block_size=8, max_requests=12)
    requests = [Request(i, [i + 1, 5], 6, allowed_tokens=(lambda g: [7 + len(g)]) if i == 9 else None) for i in range(11)]
    out = engine.run_offline(requests)
    assert out[9] == [7, 8, 9, 10, 11, 12]


def test_refused_requests(tmp_path):
    from inf_engine_b200 import Engine, Request, SamplingConfig
    d = make_model_dir(tmp_path, "tiny_a")
    engine = Engine.from_dir(d, dtype="float32", n_total_blocks=16, block_size=8, max_requests=2)
    for c, why in ((SamplingConfig(logit_bias={256: 1.0}), "outside"), (SamplingConfig(presence_penalty=float("nan")), "finite")):
        r = Request(0, [1], 2, sampling=c)
        assert not engine.submit(r) and why in r.error

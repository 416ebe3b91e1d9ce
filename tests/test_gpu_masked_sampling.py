"""What a draw may answer at the edges: masked tokens (-inf), logits that are no number, infinite ones, numbers next to 1.

The uniform number of a draw is a hash of (seed, key) and the hash can be undone, so a test names the number it wants.  Next to 1 the
walk through the tokens ends where rounding says: it must still end on a token that has a share."""

import numpy as np
import pytest
import torch

import plain_llama

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")
MODES = [("temperature", {}), ("temperature", dict(temperature=0.6)), ("top_k", dict(top_k=1500, temperature=1.2)),
         ("top_k", dict(top_k=10 ** 6)), ("top_p", dict(top_p=0.99999)), ("top_p", dict(top_p=0.5, temperature=1.4))]


def undo_splitmix64(x):
    m = (1 << 64) - 1

    def unshift(v, s):
        out = v
        for _ in range(64 // s + 1):
            out = v ^ (out >> s)
        return out
    x = unshift(x, 31) * pow(0x94D049BB133111EB, -1, 1 << 64) & m
    x = unshift(x, 27) * pow(0xBF58476D1CE4E5B9, -1, 1 << 64) & m
    return (unshift(x, 30) - 0x9E3779B97F4A7C15) & m


def seed_for(steps, key):
    """The seed that draws steps / 2^24 for the key."""
    return undo_splitmix64(undo_splitmix64(steps << 40 | 12345) ^ key)


def draw(logits, configs, keys):
    from inf_engine_b200 import kernels
    from inf_engine_b200.sampling import pack_rows
    out = torch.full((logits.shape[0],), -7, dtype=torch.int32, device=DEV)
    kernels.sample(logits.to(DEV), torch.from_numpy(pack_rows(configs, keys, logits.shape[1])).to(DEV), out)
    return out.cpu()


def near_one(mode, kw, n):
    from inf_engine_b200.sampling import SamplingConfig, uniform_of
    keys = [(i << 32) | 3 for i in range(n)]
    configs = [SamplingConfig(mode=mode, seed=seed_for((1 << 24) - 1 - i % 8, k), **kw) for i, k in enumerate(keys)]
    assert all(uniform_of(c.seed, k) == 1 - (1 + i % 8) / 2 ** 24 for i, (c, k) in enumerate(zip(configs, keys)))
    return configs, keys


@pytest.mark.parametrize("mode,kw", MODES)
@pytest.mark.parametrize("vocab,allowed,n", [(2048, 300, 1024), (40003, 6000, 96)])
def test_a_masked_token_is_never_drawn(vocab, allowed, n, mode, kw):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.full((n, vocab), -INF)
    logits[:, :allowed] = 2 * torch.randn(n, allowed, generator=g)
    configs, keys = near_one(mode, kw, n)
    out = draw(logits, configs, keys)
    assert int(out.min()) >= 0 and int(out.max()) < allowed
    for i in range(0, n, 16):
        c = configs[i]
        probs = plain_llama.filtered_distribution(logits[i], mode, c.temperature, min(c.top_k, vocab), c.top_p).double()
        assert probs[out[i]] > 0 and float(probs[:int(out[i]) + 1].sum()) >= 1 - 1e-5


@pytest.mark.parametrize("mode,kw", MODES)
@pytest.mark.parametrize("vocab", [2048, 40003])
def test_a_token_without_a_share_is_never_drawn(vocab, mode, kw):
    """exp(-300) is nothing in float32; such tokens stand at the end, where the walk would come to rest."""
    g = torch.Generator().manual_seed(vocab + 1)
    n = 512 if vocab < 10000 else 64
    logits = 2 * torch.randn(n, vocab, generator=g)
    logits[:, vocab // 2:] = -300.0
    out = draw(logits, *near_one(mode, kw, n))
    assert int(out.min()) >= 0 and int(out.max()) < vocab // 2


def rows_with(vocab, special):
    """Allowed tokens are 0 .. 99 and ``special`` stands at some of them; the others are masked."""
    g = torch.Generator().manual_seed(7)
    logits = torch.full((64, vocab), -INF)
    logits[:, :100] = torch.randn(64, 100, generator=g) - 3
    for i in range(64):
        logits[i, i], logits[i, (7 * i + 50) % 100] = special, special
    return logits


@pytest.mark.parametrize("vocab", [100, 2048, 40003])
def test_a_logit_that_is_no_number_is_never_the_answer(vocab):
    from inf_engine_b200 import kernels
    from inf_engine_b200.sampling import SamplingConfig
    logits = rows_with(vocab, NAN)
    want = torch.where(logits.isnan(), -INF, logits)
    out = torch.empty(64, dtype=torch.int32, device=DEV)
    kernels.argmax(logits.to(DEV), out)
    assert torch.equal(out.cpu().long(), want.argmax(1))
    assert torch.equal(draw(logits, [SamplingConfig()] * 64, [0] * 64).long(), want.argmax(1))
    for mode, kw in MODES:
        for steps in (0, 1 << 23, (1 << 24) - 1):
            keys = [i << 32 for i in range(64)]
            configs = [SamplingConfig(mode=mode, seed=seed_for(steps, k), **kw) for k in keys]
            got = draw(logits, configs, keys)
            for i in range(64):
                c = configs[i]
                probs = plain_llama.filtered_distribution(want[i], mode, c.temperature, min(c.top_k, vocab), c.top_p).double()
                cdf, t = probs.cumsum(0), int(got[i])
                assert probs[t] > 0, (mode, i, t)
                assert (float(cdf[t - 1]) if t else 0.0) - 1e-5 <= steps / 2 ** 24 <= float(cdf[t]) + 1e-5


@pytest.mark.parametrize("vocab", [100, 2048, 40003])
def test_an_infinite_logit_is_the_answer(vocab):
    """The first of them, whatever the mode, as when the temperature makes the largest ones infinite."""
    from inf_engine_b200.sampling import SamplingConfig
    logits = rows_with(vocab, INF)
    first = torch.tensor([min(i, (7 * i + 50) % 100) for i in range(64)], dtype=torch.int32)
    for mode, kw in [("greedy", {})] + MODES + [("top_k", dict(top_k=3, temperature=1e30)), ("temperature", dict(temperature=1e38))]:
        for steps in (0, (1 << 24) - 1):
            keys = [i << 32 for i in range(64)]
            assert torch.equal(draw(logits, [SamplingConfig(mode=mode, seed=seed_for(steps, k), **kw) for k in keys], keys), first)
    positive = logits.clamp(max=5.0) + 10
    assert torch.equal(draw(positive, [SamplingConfig(mode="temperature", temperature=1e-40)] * 64, list(range(64))), first)


@pytest.mark.parametrize("vocab", [100, 2048, 40003])
def test_masked_tokens_under_the_largest_temperature(vocab):
    """Shares become equal; a masked token still has none."""
    from inf_engine_b200.sampling import SamplingConfig
    logits = rows_with(vocab, 1.0)
    for mode, kw in (("temperature", {}), ("top_k", dict(top_k=vocab - 1)), ("top_p", dict(top_p=0.999))):
        for steps, want in ((0, 0), ((1 << 24) - 1, 99)):
            keys = [i << 32 for i in range(64)]
            got = draw(logits, [SamplingConfig(mode=mode, temperature=3e38, seed=seed_for(steps, k), **kw) for k in keys], keys)
            assert got.tolist() == [want] * 64 or (mode != "temperature" and int(got.max()) < 100)


@pytest.mark.parametrize("vocab", [100, 2048, 40003])
def test_a_row_without_a_number_answers_the_first_token(vocab):
    from inf_engine_b200 import kernels
    from inf_engine_b200.sampling import SamplingConfig
    logits = torch.full((4, vocab), -INF)
    logits[1], logits[2, 3:], logits[3, :3] = NAN, NAN, NAN
    out = torch.empty(4, dtype=torch.int32, device=DEV)
    kernels.argmax(logits.to(DEV), out)
    assert out.cpu().tolist() == [0] * 4
    for mode, kw in [("greedy", {})] + MODES:
        assert draw(logits, [SamplingConfig(mode=mode, **kw)] * 4, [0] * 4).tolist() == [0] * 4


@pytest.mark.parametrize("vocab", [100, 40003])
def test_a_temperature_that_divides_to_nothing_is_greedy(vocab):
    """Logits below 0 over 1e-40 are all -inf in float32."""
    from inf_engine_b200.sampling import SamplingConfig
    logits = -1 - torch.rand(8, vocab, generator=torch.Generator().manual_seed(3))
    for mode in ("temperature", "top_k", "top_p"):
        got = draw(logits, [SamplingConfig(mode=mode, temperature=1e-40, seed=i) for i in range(8)], list(range(8)))
        assert torch.equal(got.long(), logits.argmax(1))


@pytest.mark.parametrize("vocab", [100, 40003])
@pytest.mark.parametrize("top_p", [1e-30, 1e-46])
def test_the_largest_stays_under_the_smallest_top_p(vocab, top_p):
    """1e-46 is 0 in float32, where no mass lies below the budget."""
    from inf_engine_b200.sampling import SamplingConfig
    logits = torch.randn(16, vocab, generator=torch.Generator().manual_seed(5))
    for steps in (0, (1 << 24) - 1):
        got = draw(logits, [SamplingConfig(mode="top_p", top_p=top_p, seed=seed_for(steps, k)) for k in range(16)], list(range(16)))
        assert torch.equal(got.long(), logits.argmax(1))

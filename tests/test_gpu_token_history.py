"""Request histories and adjusted logits against plain implementations (whole numbers; 64 bits).

An adjusted logit is a chain of at most four float32 operations and the sum of the biases: with b biases of a token each step is
off by 2^-24 of its own result, so (5 + b) 2^-24 of the largest magnitude on the way bounds it.
"""

import math

import numpy as np
import pytest
import torch

from inf_engine_b200 import kernels

pytestmark = pytest.mark.gpu


def words(v):
    return -(-v // 32)


def pack(bits):
    bits = np.asarray(bits, dtype=bool)
    padded = np.zeros((bits.shape[0], words(bits.shape[1]) * 32), dtype=np.uint8)
    padded[:, :bits.shape[1]] = bits
    return np.packbits(padded, axis=1, bitorder="little").view(np.int32)


def unpack(w, v):
    return np.unpackbits(np.ascontiguousarray(w).view(np.uint8), axis=1, bitorder="little")[:, :v].astype(bool)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def plain_append(counts, bits, tokens, slots, starts, n_prompt):
    for r, slot in enumerate(slots):
        for j in range(starts[r], starts[r + 1]):
            t = tokens[j]
            if not (0 <= slot < counts.shape[0] and 0 <= t < counts.shape[1]):
                continue
            bits[slot, t] = True
            if n_prompt is None or j - starts[r] >= n_prompt[r]:
                counts[slot, t] += 1


@pytest.mark.parametrize("v", [1, 31, 32, 33, 1000, 32001])
@pytest.mark.parametrize("lengths", [[1], [0], [5, 0, 1, 700], [3] * 70, [0, 0, 2, 0]])
def test_reset_and_append(v, lengths):
    rng = np.random.default_rng(v + len(lengths))
    n_slots = 80
    counts = rng.integers(0, 3, (n_slots, v)).astype(np.int32)
    bits = rng.random((n_slots, v)) < 0.3
    bits |= counts > 0
    dc, ds = dev(counts), dev(pack(bits))
    slots = rng.permutation(n_slots)[:len(lengths)].astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    tokens = np.minimum(rng.integers(0, max(1, v // 2) + 1, starts[-1]), v - 1).astype(np.int32)
    n_prompt = np.array([rng.integers(0, n + 1) for n in lengths], dtype=np.int32)
    kernels.history_append(dc, ds, dev(tokens), dev(slots), dev(starts), dev(n_prompt))
    plain_append(counts, bits, tokens, slots, starts, n_prompt)
    assert np.array_equal(dc.cpu().numpy(), counts) and np.array_equal(ds.cpu().numpy(), pack(bits))
    some = slots[::2]
    kernels.history_reset(dc, ds, dev(some))
    counts[some] = 0
    bits[some] = False
    assert np.array_equal(dc.cpu().numpy(), counts) and np.array_equal(ds.cpu().numpy(), pack(bits))
    one = rng.integers(0, v, len(slots)).astype(np.int32)
    kernels.history_append(dc, ds, dev(one), dev(slots))
    plain_append(counts, bits, one, slots, list(range(len(slots) + 1)), None)
    assert np.array_equal(dc.cpu().numpy(), counts) and np.array_equal(ds.cpu().numpy(), pack(bits))


def test_the_same_slot_and_token_many_times_and_ids_out_of_range():
    n_slots, v = 3, 100
    counts, bits = np.zeros((n_slots, v), np.int32), np.zeros((n_slots, v), bool)
    dc, ds = dev(counts), dev(pack(bits))
    slots = np.array([1, 1, -1, 3, 2, 2 ** 31 - 1, 1], np.int32)
    tokens = np.array([7] * 5000 + [-1, 100, 31, 32, 2 ** 31 - 1, -2 ** 31, 99, 0] * 4, np.int32)
    starts = np.array([0, 2000, 4000, 4300, 4600, 5008, 5020, 5032], np.int32)
    kernels.history_append(dc, ds, dev(tokens), dev(slots), dev(starts))
    plain_append(counts, bits, tokens, slots, starts, None)
    assert np.array_equal(dc.cpu().numpy(), counts) and np.array_equal(ds.cpu().numpy(), pack(bits))
    kernels.history_reset(dc, ds, dev(np.array([2, 2, -1, 3, 2 ** 31 - 1], np.int32)))
    counts[2], bits[2] = 0, False
    assert np.array_equal(dc.cpu().numpy(), counts) and np.array_equal(ds.cpu().numpy(), pack(bits))


def case(n, v, dtype, seed, penalties=True, biases=True, masks=True, n_slots=None):
    rng = np.random.default_rng(seed)
    n_slots = n_slots or n + 2
    logits = torch.from_numpy((3 * rng.standard_normal((n, v))).astype(np.float32)).to(dtype)
    a = {"logits": logits}
    if penalties:
        counts = np.where(rng.random((n_slots, v)) < 0.1, rng.integers(1, 9, (n_slots, v)), 0).astype(np.int32)
        a["counts"], a["seen"] = counts, pack((counts > 0) | (rng.random((n_slots, v)) < 0.1))
        a["slots"] = rng.integers(-1, n_slots + 1, n).astype(np.int32)           # outside the table too: no history
        a["penalties"] = np.stack([rng.uniform(0.7, 1.5, n), rng.uniform(-1, 1, n), rng.uniform(-0.5, 0.5, n)], 1).astype(np.float32)
    if biases:
        each = rng.integers(0, 40, n)
        each[0] = 0
        a["bias_start"] = np.concatenate([[0], np.cumsum(each)]).astype(np.int32)
        a["bias_ids"] = rng.integers(-1, v + 1, a["bias_start"][-1]).astype(np.int32)
        a["bias_values"] = (5 * rng.standard_normal(a["bias_start"][-1])).astype(np.float32)
    if masks:
        m = max(1, n // 2)
        bits = rng.random((m, v)) < 0.5
        bits[0] = False                                                          # a row that may be nothing
        a["masks"] = pack(bits)
        a["mask_rows"] = rng.integers(-1, m + 1, n).astype(np.int32)
    return a


def plain_adjust(a):
    x = a["logits"].double().numpy().copy()
    n, v = x.shape
    top = np.abs(np.where(np.isfinite(x), x, 0))
    adds = np.zeros((n, v))
    for i in range(n):
        if "slots" in a and 0 <= a["slots"][i] < a["counts"].shape[0]:
            s = a["slots"][i]
            r, once, f = a["penalties"][i].astype(np.float64)
            seen = unpack(a["seen"][s:s + 1], v)[0]
            x[i] = np.where(seen, np.where(x[i] < 0, x[i] * r, x[i] / r), x[i])
            c = np.where(seen, a["counts"][s], 0)
            off = f * c + once
            top[i] = np.maximum(top[i], np.maximum(np.abs(np.where(np.isfinite(x[i]), x[i], 0)), np.abs(f * c) + abs(once)))
            x[i] = np.where(c > 0, x[i] - off, x[i])
        if "bias_ids" in a:
            for b in range(a["bias_start"][i], a["bias_start"][i + 1]):
                t = a["bias_ids"][b]
                if 0 <= t < v:
                    x[i, t] += np.float64(a["bias_values"][b])
                    adds[i, t] += 1
                    top[i, t] += abs(float(a["bias_values"][b]))
        if "masks" in a and 0 <= a["mask_rows"][i] < a["masks"].shape[0]:
            ok = unpack(a["masks"][a["mask_rows"][i]:a["mask_rows"][i] + 1], v)[0]
            x[i] = np.where(ok, x[i], -math.inf)
    return x, (5 + adds) * 2.0 ** -24 * 2 * top


def call(a, logits, out):
    t = {k: dev(v) for k, v in a.items() if k != "logits"}
    kernels.adjust_logits(logits, out, **t)


def agree(got, want, bound):
    got = got.double().cpu().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(1, 1), (1, 31), (2, 33), (3, 1000), (5, 4097), (2, 32000), (7, 50001), (70, 1024), (1, 128256)])
@pytest.mark.parametrize("parts", ["pbm", "p", "b", "m", ""])
def test_adjust(n, v, dtype, parts):
    a = case(n, v, dtype, 7 * n + v, "p" in parts, "b" in parts, "m" in parts)
    want, bound = plain_adjust(a)
    logits = a["logits"].cuda()
    out = torch.full((n, v), 9.0, device="cuda")
    before = logits.clone()
    call(a, logits, out)
    agree(out, want, bound)
    assert torch.equal(logits, before)
    if dtype is torch.float32:
        call(a, logits, logits)                                  # in place
        assert torch.equal(torch.nan_to_num(logits), torch.nan_to_num(out))


@pytest.mark.parametrize("off,pitch", [(0, 1003), (1, 1001), (4, 1012), (2, 1100)])
def test_adjust_of_slices(off, pitch):
    n, v = 6, 998
    a = case(n, v, torch.float32, off)
    want, bound = plain_adjust(a)
    src = torch.full((n, pitch), 5.0, device="cuda")
    x = src[:, off:off + v]
    x.copy_(a["logits"])
    dst = torch.full((n, pitch + 3), 5.0, device="cuda")
    y = dst[:, 3 - off % 3:3 - off % 3 + v]
    call(a, x, y)
    agree(y, want, bound)
    call(a, x, x)
    agree(x, want, bound)
    x.fill_(5.0)
    y.fill_(5.0)
    assert bool((src == 5).all()) and bool((dst == 5).all())


def test_numbers_that_are_none():
    v = 96
    a = case(4, v, torch.float32, 3, biases=False)
    a["slots"][:] = [0, 1, 2, 3]
    a["mask_rows"][:] = [-1, 1, 0, -1]
    x = a["logits"]
    x[0, ::3], x[1, ::3], x[2, ::3] = math.inf, -math.inf, math.nan
    x[3] = torch.finfo(torch.float32).min
    x[3, 1], x[3, 2] = -0.0, 0.0
    a["penalties"][3] = [1.0, 0.5, 0.25]
    with np.errstate(over="ignore", invalid="ignore"):
        want, bound = plain_adjust(a)
        want = np.where(np.abs(want) > 3.5e38, np.sign(want) * np.inf, want)
    out = torch.empty(4, v, device="cuda")
    call(a, x.cuda(), out)
    agree(out, want, bound)


def test_offsets_beyond_32_bits():
    n_slots, v = 17_000, 128_256                       # 2.2e9 counts
    counts = torch.zeros(n_slots, v, dtype=torch.int32, device="cuda")
    seen = torch.zeros(n_slots, words(v), dtype=torch.int32, device="cuda")
    slots = torch.tensor([n_slots - 1, n_slots - 2], dtype=torch.int32, device="cuda")
    tokens = torch.tensor([5, v - 1, 5, 7], dtype=torch.int32, device="cuda")
    kernels.history_append(counts, seen, tokens, slots, torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda"))
    assert int(counts[-1, 5]) == 2 and int(counts[-1, v - 1]) == 1 and int(counts[-2, 7]) == 1 and int(counts.sum(dtype=torch.int64)) == 4
    m = 17_000
    logits = torch.ones(m, v, device="cuda")
    at = torch.full((m,), -1, dtype=torch.int32, device="cuda")
    at[-1] = n_slots - 1
    pen = torch.tensor([[2.0, 0.25, 0.5]], device="cuda").repeat(m, 1)
    kernels.adjust_logits(logits, logits, at, pen, counts, seen)
    assert logits[-1, 5].item() == 0.5 - 1.25 and logits[-1, v - 1].item() == 0.5 - 0.75
    assert int((logits != 1).sum()) == 2
    kernels.history_reset(counts, seen, slots)
    assert int(counts.sum(dtype=torch.int64)) == 0 and int(seen.sum(dtype=torch.int64)) == 0


def test_captured_with_the_history_that_moves_on():
    n, v, n_slots = 4, 5000, 6
    a = case(n, v, torch.float32, 5, biases=False, masks=False, n_slots=n_slots)
    a["slots"] = np.array([5, 0, 3, 1], np.int32)
    logits, out = a["logits"].cuda(), torch.empty(n, v, device="cuda")
    counts, seen, slots, pen = dev(a["counts"]), dev(a["seen"]), dev(a["slots"]), dev(a["penalties"])
    tokens = torch.zeros(n, dtype=torch.int32, device="cuda")

    def step():
        kernels.adjust_logits(logits, out, slots, pen, counts, seen)
        kernels.argmax(out, tokens)
        kernels.history_append(counts, seen, tokens, slots)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    kernels.core()
    with torch.cuda.graph(graph, stream=side):
        step()
    bits = unpack(a["seen"], v)
    for _ in range(12):
        graph.replay()
        want, bound = plain_adjust(a)
        agree(out, want, bound)
        got = tokens.cpu().numpy()
        assert np.array_equal(got, out.cpu().numpy().argmax(1))
        plain_append(a["counts"], bits, got, a["slots"], list(range(n + 1)), None)
        a["seen"] = pack(bits)
    assert np.array_equal(counts.cpu().numpy(), a["counts"]) and np.array_equal(seen.cpu().numpy(), a["seen"])

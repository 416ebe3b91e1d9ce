"""Lists of biases of any length, naming tokens once or many times, in any order: bit for bit the sums in the list's order, in float32, and a
time in proportion to the list."""

import numpy as np
import pytest
import torch

from inf_engine_b200 import kernels

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def plain(logits, lists, masks=None):
    out = logits.copy()
    for i, (ids, values) in enumerate(lists):
        sums = {}
        for t, v in zip(ids.tolist(), values):
            if 0 <= t < logits.shape[1]:
                sums[t] = np.float32(sums.get(t, np.float32(0)) + v)
        for t, s in sums.items():
            out[i, t] = np.float32(out[i, t] + s)
        if masks is not None and masks[i] is not None:
            out[i, ~masks[i]] = -np.inf
    return out


def call(logits, lists, masks=None, in_place=False, dtype=torch.float32):
    start = np.concatenate([[0], np.cumsum([len(i) for i, _ in lists])]).astype(np.int32)
    ids = np.concatenate([i for i, _ in lists]).astype(np.int32)
    values = np.concatenate([v for _, v in lists]).astype(np.float32)
    kw = dict(bias_start=dev(start), bias_ids=dev(ids), bias_values=dev(values))
    if masks is not None:
        given = [m for m in masks if m is not None]
        v = logits.shape[1]
        bits = np.zeros((len(given), -(-v // 32) * 32), bool)
        bits[:, :v] = given
        rows = np.full(len(masks), -1, np.int32)
        rows[[i for i, m in enumerate(masks) if m is not None]] = np.arange(len(given))
        kw.update(mask_rows=dev(rows), masks=dev(np.packbits(bits, axis=1, bitorder="little").view(np.int32)))
    x = dev(logits).to(dtype)
    out = x if in_place else torch.empty(x.shape, device="cuda")
    kernels.adjust_logits(x, out, **kw)
    return out.cpu().numpy()


LENGTHS = [0, 1, 2, 31, 32, 33, 127, 128, 129, 500, 3000]


@pytest.mark.parametrize("kind", ["distinct", "any", "few tokens", "one token", "sorted", "outside"])
@pytest.mark.parametrize("v", [1, 33, 1000, 4097, 50001])
def test_sums_in_the_lists_order(v, kind):
    rng = np.random.default_rng(v)
    lists = []
    for n in LENGTHS:
        if kind == "distinct":
            ids = rng.permutation(v)[:n]
        elif kind == "sorted":
            ids = np.sort(rng.integers(0, v, n))
        elif kind == "few tokens":
            ids = rng.choice(rng.integers(0, v, 5), n)
        elif kind == "one token":
            ids = np.full(n, v - 1)
        else:
            ids = rng.integers(-5 if kind == "outside" else 0, v + (40 if kind == "outside" else 0), n)
            if kind == "outside" and n:
                ids[rng.integers(0, n, 3)] = [-2 ** 31, 2 ** 31 - 1, v]
        lists.append((ids.astype(np.int64), (rng.standard_normal(len(ids)) * 10.0 ** rng.integers(-3, 4, len(ids))).astype(np.float32)))
    logits = rng.standard_normal((len(LENGTHS), v)).astype(np.float32)
    masks = [None if i % 3 == 0 else rng.random(v) < 0.5 for i in range(len(LENGTHS))]
    for m in (None, masks):
        want = plain(logits, lists, m)
        for in_place in (False, True):
            assert np.array_equal(call(logits, lists, m, in_place), want)
    half = torch.from_numpy(logits).to(torch.bfloat16).float().numpy()
    assert np.array_equal(call(half, lists, dtype=torch.bfloat16), plain(half, lists))


def test_numbers_that_are_none_and_zeros():
    logits = np.array([[1.0, -0.0, np.inf, 2.0, 0.0, 3.0]] * 2, np.float32)
    ids = np.array([0, 1, 2, 0, 3, 2] * 40)
    values = np.array([np.nan, -0.0, -np.inf, 1.0, np.inf, 1.0] * 40, np.float32)
    lists = [(ids, values), (np.zeros(0, np.int64), np.zeros(0, np.float32))]
    with np.errstate(invalid="ignore"):
        want = plain(logits, lists)
    got = call(logits, lists)
    assert np.array_equal(got, want, equal_nan=True) and np.isnan(got[0, [0, 2]]).all() and got[0, 3] == np.inf


@pytest.mark.parametrize("v", [128256])
@pytest.mark.parametrize("kind", ["every token", "one token behind many that are none"])
def test_time_in_proportion_to_the_list(v, kind):
    """0.6 ms for each here; when every bias looked through the list it was 119 ms for every token of a vocabulary."""
    if kind == "every token":
        ids = torch.arange(v, dtype=torch.int32, device="cuda")
    else:
        ids = torch.cat([torch.full((200000,), -1, dtype=torch.int32, device="cuda"), torch.full((200000,), 7, dtype=torch.int32, device="cuda")])
    values = torch.ones(ids.shape[0], device="cuda")
    start = torch.tensor([0, ids.shape[0]], dtype=torch.int32, device="cuda")
    x = torch.zeros(1, v, device="cuda")
    out = torch.empty_like(x)
    times = []
    for _ in range(3):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        kernels.adjust_logits(x, out, bias_start=start, bias_ids=ids, bias_values=values)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    if kind == "every token":
        assert bool((out == 1).all())
    else:
        assert float(out[0, 7]) == 200000 and float(out.sum()) == 200000
    assert min(times) < 20, times


def test_one_list_for_many_rows_and_a_row_alone():
    """Rows may share stretches of the list, and a start beyond it ends there."""
    v = 5000
    rng = np.random.default_rng(3)
    ids, values = rng.integers(0, v, 600).astype(np.int32), rng.standard_normal(600).astype(np.float32)
    logits = rng.standard_normal((4, v)).astype(np.float32)
    out = torch.empty(4, v, device="cuda")
    kernels.adjust_logits(dev(logits), out, bias_start=dev(np.array([-9, 300, 200, 600, 900], np.int32)), bias_ids=dev(ids), bias_values=dev(values))
    cuts = [(0, 300), (300, 200), (200, 600), (600, 600)]
    want = plain(logits, [(ids[a:b].astype(np.int64), values[a:b]) for a, b in cuts])
    assert np.array_equal(out.cpu().numpy(), want)

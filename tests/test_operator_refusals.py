"""What the 8-bit products, request histories and adjusted logits refuse, before anything reaches a GPU."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from inf_engine_b200 import kernels
from inf_engine_b200.kernels import KernelError

FP8 = torch.float8_e4m3fn


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def codes(m, k):
    return kernels.fp8_empty(m, k, "cpu")


def refused(why, fn, *args, **kw):
    with pytest.raises(KernelError, match=why):
        fn(*args, **kw)


def test_quantisers():
    x, q, s = torch.zeros(4, 200), codes(4, 200), torch.zeros(4, 2)
    refused("float32 or bfloat16", kernels.fp8_quantize_rows, x.half(), q, s)
    refused("float32 or bfloat16", kernels.fp8_quantize_rows, x[0], q, s)
    refused("columns of x are adjacent", kernels.fp8_quantize_rows, torch.zeros(4, 400)[:, ::2], q, s)
    refused("float8_e4m3fn", kernels.fp8_quantize_rows, x, q.view(torch.uint8), s)
    refused("16 bytes", kernels.fp8_quantize_rows, x, torch.zeros(4, 200, dtype=torch.uint8).view(FP8), s)
    refused("16 bytes", kernels.fp8_quantize_rows, x, codes(4, 208)[:, 3:203], s)
    refused("another shape", kernels.fp8_quantize_rows, x, codes(4, 199), s)
    refused("scales is", kernels.fp8_quantize_rows, x, q, torch.zeros(4, 1))
    refused("scales is", kernels.fp8_quantize_rows, x, q, s.double())
    refused("scales is", kernels.fp8_quantize_blocks, x, q, s)
    refused("contiguous", kernels.fp8_quantize_blocks, torch.zeros(300, 200), codes(300, 200), torch.zeros(2, 3).t())
    refused("current device", kernels.fp8_quantize_rows, x, q, s)
    refused("current device", kernels.fp8_quantize_blocks, x, q, torch.zeros(1, 2))


def test_product():
    x, w, sw, out = torch.zeros(3, 200), codes(130, 200), torch.ones(2, 2), torch.zeros(3, 130)
    q, sx = codes(3, 200), torch.ones(3, 2)
    g = kernels.gemm_fp8
    refused("w is a float8", g, x, torch.zeros(130, 200), sw, out)
    refused("x is \\[m, k\\]", g, torch.zeros(3, 199), w, sw, out)
    refused("x is \\[m, k\\]", g, x, w, sw, torch.zeros(3, 131))
    refused("out is", g, x, w, sw, out.half())
    refused("out is", g, x, w, sw, torch.zeros(130, 3).t())
    refused("out is", g, x, w, sw, torch.zeros(1, 130).expand(3, 130))
    refused("w_scales", g, x, w, torch.ones(2, 1), out)
    refused("w_scales", g, x, w, torch.ones(2, 2, dtype=torch.bfloat16), out)
    refused("w_scales", g, x, w, torch.ones(2, 2).t(), out) if not torch.ones(2, 2).t().is_contiguous() else None
    refused("codes of x come with", g, q, w, sw, out)
    refused("codes of x come with", g, q, w, sw, out, torch.ones(3, 1))
    refused("x_scales go with", g, x, w, sw, out, sx)
    refused("16 bytes", g, torch.zeros(3, 200, dtype=torch.uint8).view(FP8), w, sw, out, sx)
    refused("k is 0", g, torch.zeros(3, 0), codes(130, 0), torch.ones(2, 0), out)
    refused("current device", g, x, w, sw, out)
    refused("current device", g, q, w, sw, out, sx)
    one = torch.zeros(1, 200, dtype=torch.uint8).view(FP8)                # one row needs no room behind it
    refused("current device", g, one, w, sw, out[:1], sx[:1])


def test_history():
    counts, seen = i32(4, 100), i32(4, 4)
    a = kernels.history_append
    refused("counts is", kernels.history_reset, counts.long(), seen, i32(1))
    refused("seen is", kernels.history_reset, counts, i32(4, 3), i32(1))
    refused("slots is", kernels.history_reset, counts, seen, i32(2, 1))
    refused("contiguous int32 vectors", a, counts, seen, torch.zeros(3), i32(3))
    refused("one token a slot", a, counts, seen, i32(3), i32(2))
    refused("starts is", a, counts, seen, i32(3), i32(2), i32(2))
    refused("n_prompt is", a, counts, seen, i32(3), i32(2), i32(3), i32(3))
    refused("current device", a, counts, seen, i32(3), i32(3))
    refused("current device", kernels.history_reset, counts, seen, i32(3))


def test_adjust():
    f = kernels.adjust_logits
    x, out = torch.zeros(3, 100), torch.zeros(3, 100)
    p = dict(slots=i32(3), penalties=torch.ones(3, 3), counts=i32(4, 100), seen=i32(4, 4))
    b = dict(bias_start=i32(4), bias_ids=i32(5), bias_values=torch.zeros(5))
    m = dict(mask_rows=i32(3), masks=i32(2, 4))
    refused("float32 and bfloat16|out is", f, x, out.half())
    refused("out is float32", f, x, out.bfloat16())
    refused("adjacent columns", f, x, torch.zeros(3, 99))
    refused("adjacent columns", f, torch.zeros(100, 3).t(), out)
    refused("rows overlap", f, torch.zeros(1, 100).expand(3, 100), out)
    buf = torch.zeros(1000)
    refused("shares memory", f, buf[:300].view(3, 100), buf[8:308].view(3, 100))
    refused("shares memory", f, torch.as_strided(buf, (3, 100), (150, 1)), torch.as_strided(buf, (3, 100), (150, 1), 60))
    refused("shares memory", f, buf.view(torch.bfloat16)[:300].view(3, 100), buf[:300].view(3, 100))
    for names, whole in ((p, "penalties need"), (b, "biases need"), (m, "masks need")):
        for gone in names:
            refused(whole, f, x, out, **{k: v for k, v in names.items() if k != gone})
    refused("another vocabulary", f, x, out, **{**p, "counts": i32(4, 99)})
    refused("seen is", f, x, out, **{**p, "seen": i32(4, 5)})
    refused("slots is", f, x, out, **{**p, "slots": i32(2)})
    refused("penalties is", f, x, out, **{**p, "penalties": torch.ones(3, 2)})
    refused("bias_start is", f, x, out, **{**b, "bias_start": i32(3)})
    refused("bias_values is", f, x, out, **{**b, "bias_values": torch.zeros(4)})
    refused("mask_rows is", f, x, out, **{**m, "mask_rows": i32(2)})
    refused("masks is", f, x, out, **{**m, "masks": i32(2, 3)})
    refused("current device", f, x, out, **p, **b, **m)
    # side by side in one buffer is no overlap: the refusal is the device's
    refused("current device", f, torch.as_strided(buf, (3, 100), (250, 1)), torch.as_strided(buf, (3, 100), (250, 1), 120))


@pytest.mark.parametrize("name,high", [("fp8_quantize_rows", 1), ("fp8_quantize_blocks", 128)])
def test_codes_lie_apart_from_what_they_come_from(name, high):
    f = getattr(kernels, name)
    buf = torch.zeros(4 * 1024, dtype=torch.uint8)
    scales = torch.zeros(-(-4 // high), 2)
    x = buf.view(torch.bfloat16)[:4 * 200].view(4, 200)
    codes = buf.view(kernels.FP8)
    refused("shares memory", f, x, torch.as_strided(codes, (4, 200), (208, 1)), scales)
    refused("shares memory", f, x, torch.as_strided(codes, (4, 200), (208, 1), 16 * 99), scales)     # x ends behind 1,600 bytes
    refused("current device", f, x, torch.as_strided(codes, (4, 200), (208, 1), 1600), scales)
    refused("current device", f, buf.view(torch.float32)[:800].view(4, 200)[:0], torch.as_strided(codes, (4, 200), (208, 1))[:0], scales[:0])
    # side by side in rows of 1,024 bytes
    rows = torch.as_strided(buf.view(torch.bfloat16), (4, 200), (512, 1))
    refused("current device", f, rows, torch.as_strided(codes, (4, 200), (1024, 1), 512), scales)
    refused("shares memory", f, rows, torch.as_strided(codes, (4, 200), (1024, 1), 384), scales)


SIZES = """
from inf_engine_b200 import kernels
big, bad_size = 1 << 31, -2
def words(pack, n, at):
    return pack(*[big if i == at else 1 for i in range(n)])
fp8, core = kernels.fp8_library(), kernels.core()
for at in (4, 5):
    assert fp8.ie_fp8_quantize_rows(words(kernels._11_words, 11, at)) == bad_size
    assert fp8.ie_fp8_quantize_blocks(words(kernels._9_words, 9, at)) == bad_size
for at in (7, 8, 9):
    assert fp8.ie_gemm_fp8(words(kernels._18_words, 18, at)) == bad_size
for at in (3, 4, 5):
    assert core.ie_history_reset(words(kernels._7_words, 7, at)) == bad_size
for at in (6, 7, 8, 9):
    assert core.ie_history_append(words(kernels._11_words, 11, at)) == bad_size
for at in (12, 13, 16, 17, 18):
    assert core.ie_adjust_logits(words(kernels._21_words, 21, at)) == bad_size
"""


def test_launchers_refuse_sizes_that_pass_32_bits():
    """Before anything is launched, so this runs without a GPU; in a process of its own, which loads the libraries."""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", SIZES], cwd=root, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]

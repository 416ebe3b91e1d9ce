"""Memory that a call writes lies apart from its other arguments, scales and tables included: every layout in which the bytes meet is
refused, and columns of one buffer, side by side, are not.  The launchers decide it from addresses and strides alone, so this runs without a
GPU, over made-up addresses; in a process of its own, which sees no device, so that nothing can be launched."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

PRELUDE = """
import random
from inf_engine_b200 import kernels
fp8, core = kernels.fp8_library(), kernels.core()
OVERLAP = -6
A = 1 << 20
def matrix(at, rows, cols, row, col, size):
    return {at + size * (i * row + j * col) + b for i in range(rows) for j in range(cols) for b in range(size)}
"""

QUANTISERS = PRELUDE + """
rng = random.Random(1)
seen = {True: 0, False: 0}
for case in range(1200):
    blocks = case % 2
    rows, cols, dtype = rng.randint(1, 300 if blocks else 9), rng.randint(1, 400), rng.randint(0, 1)
    size, groups = (4, 2)[dtype], -(-cols // 128)
    srows = -(-rows // 128) if blocks else rows
    side = rng.random() < 0.4          # x, codes and scales as columns of one buffer
    if side:
        pitch = 16 * rng.randint(-(-(cols * size + cols + 4 * groups) // 16), 200)
        x, ldx, ldc = A, pitch // size, pitch
        codes = A + 16 * rng.randint(-(-cols * size // 16), max(-(-cols * size // 16), (pitch - cols) // 16))
        if blocks:
            s_row, s_col = groups, 1
        else:
            s_row, s_col = pitch // 4, 1
        scales = A + 4 * rng.randint(0, pitch // 4)
    else:
        ldx, ldc = cols + rng.randint(0, 9), 16 * (-(-cols // 16) + rng.randint(0, 2))
        x = A + 16 * rng.randint(0, 400)
        codes = x + 16 * (rows * ldx * size // 16 + 1)
        s_row, s_col = (groups, 1) if blocks else rng.choice([(groups, 1), (1, rows), (groups + 3, 1), (2 * groups, 2), (1, rows + 5)])
        end = codes + rows * ldc
        scales = rng.choice([A - 4 * rng.randint(1, 3000), end + 4 * rng.randint(-30, 30) // 4 * 4, x + 4 * rng.randint(-40, rows * ldx * size // 4)]) // 4 * 4
    b = {"x": matrix(x, rows, cols, ldx, 1, size), "codes": matrix(codes, rows, cols, ldc, 1, 1), "scales": matrix(scales, srows, groups, s_row, s_col, 4)}
    meets = bool(b["scales"] & (b["x"] | b["codes"]))
    if blocks:
        rc = fp8.ie_fp8_quantize_blocks(kernels._9_words(x, dtype, codes, scales, rows, cols, ldx, ldc, 0))
    else:
        rc = fp8.ie_fp8_quantize_rows(kernels._11_words(x, dtype, codes, scales, rows, cols, ldx, ldc, s_row, s_col, 0))
    if meets:
        assert rc == OVERLAP, (case, rows, cols)
    far = min(b["scales"]) > max(b["x"] | b["codes"]) or max(b["scales"]) < min(b["x"] | b["codes"])
    if far or (side and not blocks and not meets):
        assert rc != OVERLAP, (case, rows, cols)
    seen[meets] += 1
assert min(seen.values()) > 150, seen
"""

PRODUCT = PRELUDE + """
rng = random.Random(2)
seen = {True: 0, False: 0}
for case in range(1000):
    m, n, k = rng.randint(1, 40), rng.randint(1, 300), rng.randint(1, 400)
    kb, nb, dtype, coded = -(-k // 128), -(-n // 128), rng.randint(0, 1), rng.random() < 0.5
    size = (4, 2)[dtype]
    ldy = n + rng.randint(0, 5)
    out = A
    end = (out + size * m * ldy + 15) // 16 * 16
    sw = rng.choice([end, A - 4 * kb * nb - 64, A + 4 * rng.randint(-kb * nb - 2, size * m * ldy // 4 + 2)])
    s_row, s_col = rng.choice([(kb, 1), (1, m), (0, 1), (kb + 2, 1)])
    sx = rng.choice([end + 4096, A - (1 << 16), A + 4 * rng.randint(-kb * m - 2, size * m * ldy // 4 + 2)]) if coded else 0
    room = (end if rng.random() < 0.3 else end + (1 << 14)) if not coded else 0
    bytes_ = m * (-(-k // 16) * 16 + 4 * kb) if room else 0
    x, w = A + (1 << 24), A + (1 << 25)
    b_out, b_sw = matrix(out, m, n, ldy, 1, size), matrix(sw, nb, kb, kb, 1, 4)
    b_sx = matrix(sx, m, kb, s_row, s_col, 4) if coded else set()
    b_room = set(range(room, room + bytes_))
    meets = bool((b_out | b_room) & (b_sw | b_sx))
    rc = fp8.ie_gemm_fp8(kernels._18_words(x, 2 if coded else 1, sx, w, sw, out, dtype, m, n, k, 512, s_row, s_col, 512, ldy, room, bytes_, 0))
    if meets:
        assert rc == OVERLAP, case
    if all(not q or min(q) > max(b_out) or max(q) < min(b_out) for q in (b_sw, b_sx)) and not meets:
        assert rc != OVERLAP, case
    seen[meets] += 1
assert min(seen.values()) > 150, seen
"""

PLACES = PRELUDE + """
rng = random.Random(3)
seen = {True: 0, False: 0}
for case in range(3000):
    rows, groups, s_row, s_col = rng.randint(1, 7), rng.randint(1, 7), rng.randint(0, 9), rng.randint(0, 9)
    places = [i * s_row + j * s_col for i in range(rows) for j in range(groups)]
    shared = len(set(places)) < len(places)
    cols = 128 * groups - rng.randint(0, 127)
    rc = fp8.ie_fp8_quantize_rows(kernels._11_words(A, 1, A + (1 << 20), A + (1 << 22), rows, cols, cols, 1024, s_row, s_col, 0))
    assert (rc == -7) == shared, (case, rows, groups, s_row, s_col)
    seen[shared] += 1
assert min(seen.values()) > 500, seen
"""

TABLES = PRELUDE + """
# every argument has its own place, and every one that is written is then moved over every other one's first and last word
def check(call, pack, layout, words, written):
    # layout: name -> (index of the address, number of words); words: the arguments, addresses included
    at = {}
    place = A
    for name, (i, n) in layout.items():
        at[name] = words[i] = place
        place += 4 * n
    assert call(pack(*words)) != OVERLAP
    for w in written:
        for name, (i, n) in layout.items():
            if name == w:
                continue
            iw, nw = layout[w]
            for moved, refused in ((at[name] - 4 * nw, False), (at[name] - 4 * nw + 4, True), (at[name] + 4 * n - 4, True), (at[name] + 4 * n, False)):
                other = list(words)
                for j, (k, _) in enumerate(layout.values()):
                    if k != i:
                        other[k] = A * 100 + (j << 30)        # the others far away
                other[iw] = moved
                rc = call(pack(*other))
                assert (rc == OVERLAP) == refused, (call.__name__, w, name, moved - at[name])
v, bits, slots, n, tokens, masks, biases = 1000, 32, 5, 3, 40, 4, 17
check(core.ie_history_reset, kernels._7_words, {"counts": (0, slots * v), "seen": (1, slots * bits), "slots": (2, n)},
      [0, 0, 0, n, slots, v, 0], ("counts", "seen"))
check(core.ie_history_append, kernels._11_words,
      {"counts": (0, slots * v), "seen": (1, slots * bits), "tokens": (2, tokens), "slots": (3, n), "starts": (4, n + 1), "n_prompt": (5, n)},
      [0] * 6 + [tokens, n, slots, v, 0], ("counts", "seen"))
layout = {"out": (2, n * v), "slots": (3, n), "penalties": (4, 3 * n), "counts": (5, slots * v), "seen": (6, slots * bits), "bias_start": (7, n + 1),
          "bias_ids": (8, biases), "bias_values": (9, biases), "mask_rows": (10, n), "masks": (11, masks * bits)}
check(core.ie_adjust_logits, kernels._21_words, layout, [A * 1000, 0] + [0] * 10 + [n, v, v, v, slots, biases, masks, 0, 0], ("out",))
# a table between the rows of out
words = [A * 1000, 0, A] + [0] * 9 + [n, v, v, v + 50, slots, biases, masks, 0, 0]
for gap, refused in ((0, False), (18, False), (19, True), (-1, True)):
    words[11] = A + 4 * (v + gap)                           # 32 words of one mask in a gap of 50
    words[18] = 1
    rc = core.ie_adjust_logits(kernels._21_words(*words))
    assert (rc == OVERLAP) == refused, gap
"""


def run(program):
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=900,
                       env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 0, r.stderr[-2000:]


def test_scales_of_the_quantisers():
    run(QUANTISERS)


def test_scales_of_the_product():
    run(PRODUCT)


def test_each_scale_has_its_place():
    run(PLACES)


def test_tables_of_histories_and_logits():
    run(TABLES)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5])
def test_scales_beside_their_codes_and_over_them(n):
    from inf_engine_b200 import kernels
    from test_gpu_fp8 import codes_of, rows, same
    x = rows(n, 300, torch.bfloat16, n)
    buf = torch.zeros(n, 352, dtype=torch.uint8, device="cuda")                # a row: 300 codes, room to 320, three scales
    codes, scales = buf.view(kernels.FP8)[:, :300], buf.view(torch.float32)[:, 80:83]
    kernels.fp8_quantize_rows(x, codes, scales)
    want, ws = codes_of(x)
    assert same(codes, want) and torch.equal(scales.double(), ws)
    with pytest.raises(kernels.KernelError, match="shared with another argument"):
        kernels.fp8_quantize_rows(x, codes, buf.view(torch.float32)[:, 74:77])
    with pytest.raises(kernels.KernelError, match="shared with another argument"):
        kernels.fp8_quantize_rows(x, codes, x.view(torch.float32)[:, 10:13])
    with pytest.raises(kernels.KernelError, match="shared with another argument"):
        kernels.fp8_quantize_blocks(x, codes, x.view(torch.float32).view(-1)[:3].view(1, 3))
    w = kernels.fp8_empty(130, 300, "cuda")
    sw = torch.ones(2, 3, device="cuda")
    kernels.fp8_quantize_blocks(rows(130, 300, torch.bfloat16, 3), w, sw)
    out = torch.empty(n * 130 + 6, device="cuda")
    kernels.gemm_fp8(codes, w, sw, out[:n * 130].view(n, 130), scales)
    for over in (dict(w_scales=out[-9:-3].view(2, 3), x_scales=scales), dict(w_scales=sw, x_scales=out[:3].expand(n, 3))):
        with pytest.raises(kernels.KernelError, match="shared with another argument"):
            kernels.gemm_fp8(codes, w, out=out[:n * 130].view(n, 130), **over)
    room = torch.empty(8192, dtype=torch.uint8, device="cuda")
    with pytest.raises(kernels.KernelError, match="shared with another argument"):
        kernels.gemm_fp8(x, w, room[-24:].view(torch.float32).view(2, 3), out[:n * 130].view(n, 130), scratch=room)


@pytest.mark.gpu
def test_expanded_scales_are_refused_as_an_output():
    from inf_engine_b200 import kernels
    from test_gpu_fp8 import codes_of, rows
    x = rows(4, 300, torch.bfloat16, 1)
    codes, one = kernels.fp8_empty(4, 300, "cuda"), torch.zeros(1, 3, device="cuda")
    with pytest.raises(kernels.KernelError, match="share a place"):
        kernels.fp8_quantize_rows(x, codes, one.expand(4, 3))
    woven = torch.zeros(64, device="cuda").as_strided((4, 3), (2, 9))          # odd, but each has its own
    kernels.fp8_quantize_rows(x, codes, woven)
    assert torch.equal(woven.double(), codes_of(x)[1])


@pytest.mark.gpu
def test_tables_over_what_is_written_are_refused():
    from inf_engine_b200 import kernels
    i32 = dict(dtype=torch.int32, device="cuda")
    counts, seen = torch.zeros(3, 64, **i32), torch.zeros(3, 2, **i32)
    one = torch.zeros(1, **i32)
    for call in (lambda: kernels.history_reset(counts, counts.view(-1)[:6].view(3, 2), one), lambda: kernels.history_reset(counts, seen, seen[1, :1]),
                 lambda: kernels.history_append(counts, seen, counts[0, :1], one), lambda: kernels.history_append(counts, seen, one, seen[2, 1:])):
        with pytest.raises(kernels.KernelError, match="shared with another argument"):
            call()
    logits = torch.zeros(3, 64, device="cuda")
    with pytest.raises(kernels.KernelError, match="shared with another argument"):
        kernels.adjust_logits(logits, logits, mask_rows=torch.zeros(3, **i32), masks=logits.view(torch.int32)[:1, :2])
    kernels.history_append(counts, seen, one, one)
    kernels.history_reset(counts, seen, one)
    assert not bool(counts.any()) and not bool(seen.any())

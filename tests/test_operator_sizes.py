"""Sizes next to 2^31: what rounds them up (to blocks of 128 columns, 4,096 logits, 256 tokens) stays within 32 bits, because launchers refuse
what is above their limit.  Before anything is launched, so this runs without a GPU; in a process of its own, which loads the libraries."""

import subprocess
import sys
from pathlib import Path

SIZES = """
from inf_engine_b200 import kernels
most, bad_size = 0x7f000000, -2
fp8, core = kernels.fp8_library(), kernels.core()
entries = ((fp8.ie_fp8_quantize_rows, kernels._11_words, 11, (4, 5)), (fp8.ie_fp8_quantize_blocks, kernels._9_words, 9, (4, 5)),
           (fp8.ie_gemm_fp8, kernels._18_words, 18, (7, 8, 9)), (core.ie_history_reset, kernels._7_words, 7, (3, 4, 5)),
           (core.ie_history_append, kernels._11_words, 11, (6, 7, 8, 9)), (core.ie_adjust_logits, kernels._21_words, 21, (12, 13, 16, 17, 18)))
for call, pack, n, sizes in entries:
    for at in sizes:
        # the other sizes are 0, so that what is admitted has nothing to do
        assert call(pack(*[most if i == at else 0 for i in range(n)])) == 0, (call.__name__, at)
        for size in (most + 1, (1 << 31) - 256, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 1, -1, -(1 << 31)):
            assert call(pack(*[size if i == at else 1 for i in range(n)])) == bad_size, (call.__name__, at, size)
"""


def test_launchers_refuse_sizes_without_room_to_round_up():
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", SIZES], cwd=root, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]

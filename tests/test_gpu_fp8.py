"""The 8-bit quantisers and their product against the definition in 64 bits.

Bounds.  A code is one rounding to e4m3 of a number that a power of two scales exactly, so codes and scales are compared bit for
bit.  A product's block of 128 columns is four steps of 32 products on the tensor cores, whose 33 addends may each lose a unit in
the last place of the largest: at most 4 * 33 * 2^-23 of the sum S of the terms' magnitudes; adding the scaled blocks rounds twice
a block, 2 (K / 128) * 2^-24 of S.  A bfloat16 result adds half a step, 2^-8 of itself.
"""

import pytest
import torch

from inf_engine_b200 import kernels

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def codes_of(x, high=1):
    """(code values, scales) in float64, by the definition: groups of ``high`` rows x 128 columns."""
    m, k = x.shape
    mb, kb = -(-m // high), -(-k // 128)
    p = torch.zeros(mb * high, kb * 128, dtype=torch.float64, device=x.device)
    p[:m, :k] = x.double()
    p = p.view(mb, high, kb, 128)
    bad = ~torch.isfinite(p)
    top = torch.where(bad, 0.0, p.abs()).amax(dim=(1, 3))
    e = torch.full_like(top, -126.0)
    while bool((top > 448 * torch.exp2(e)).any()):
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
    scale = torch.where(top > 0, torch.exp2(e), 1.0)
    q = p / scale[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.where(bad, float("nan"), torch.round(q / step) * step)
    return q.view(mb * high, kb * 128)[:m, :k], scale


def rows(m, k, dtype, seed=0, wide=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    if wide:
        x = x * torch.exp(3 * torch.randn(m, 1, generator=g, device="cuda"))
    return x.to(dtype)


def quantized(x, high=1):
    codes = kernels.fp8_empty(*x.shape, x.device)
    scales = torch.empty(-(-x.shape[0] // high), -(-x.shape[1] // 128), device=x.device)
    (kernels.fp8_quantize_rows if high == 1 else kernels.fp8_quantize_blocks)(x, codes, scales)
    return codes, scales


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=1e9), torch.nan_to_num(b, nan=1e9))


def expect(x, sx, w, sw):
    """(exact product, sum of the terms' magnitudes), float64, of codes and scales."""
    k = x.shape[1]
    n = w.shape[0]
    xv = x.double() * sx.double().repeat_interleave(128, 1)[:, :k]
    wv = w.double() * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return xv @ wv.t(), xv.abs() @ wv.abs().t()


def check_product(out, want, mag, k):
    bound = (4 * 33 * 2.0 ** -23 + 2 * (-(-k // 128)) * 2.0 ** -24) * mag
    if out.dtype is torch.bfloat16:
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
    worst = ((out.double() - want).abs() - bound).max()
    assert float(worst) <= 0, f"off by {float(worst)} more than the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 127), (3, 128), (5, 129), (7, 2048), (33, 1000), (300, 264), (2, 8200)])
def test_rows(shape, dtype):
    x = rows(*shape, dtype)
    codes, scales = quantized(x)
    want, ws = codes_of(x)
    assert same(codes, want) and torch.equal(scales.double(), ws)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (127, 130), (128, 128), (129, 257), (1000, 2040), (300, 64)])
def test_blocks(shape, dtype):
    x = rows(*shape, dtype)
    codes, scales = quantized(x, 128)
    want, ws = codes_of(x, 128)
    assert same(codes, want) and torch.equal(scales.double(), ws)


@pytest.mark.parametrize("high", [1, 128])
def test_numbers_at_the_borders(high):
    top = 448.0
    x = torch.zeros(9, 384, device="cuda")
    x[1, 5] = top
    x[2, 5] = torch.nextafter(torch.tensor(top), torch.tensor(1e9))
    x[3, 130] = 1.75 * 2.0 ** 127
    x[3, 131] = torch.finfo(torch.float32).max
    x[4] = torch.finfo(torch.float32).tiny / 8          # subnormal
    x[5, :128] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0] * 32)
    x[6, 256:] = float("inf")
    x[7, 0] = -3.0
    x[8] = torch.linspace(-500, 500, 384)
    for i in range(9):
        one = x[i:i + 1]
        codes, scales = quantized(one, high)
        want, ws = codes_of(one, high)
        assert same(codes, want) and torch.equal(scales.double(), ws), i


def test_rows_of_other_strides():
    buf = rows(20, 700, torch.bfloat16)
    for x in (buf[:, 3:203], buf[::2, 8:400], buf[:, :1], buf[:1].expand(6, 700)):
        codes_buf = torch.full((x.shape[0], 1024), 3, dtype=torch.uint8, device="cuda")
        codes = codes_buf[:, 16:16 + x.shape[1]].view(FP8)
        scales = torch.empty(-(-x.shape[1] // 128), x.shape[0], device="cuda").t()
        kernels.fp8_quantize_rows(x, codes, scales)
        want, ws = codes_of(x)
        assert same(codes, want) and torch.equal(scales.double(), ws)
        assert int((codes_buf[:, :16] != 3).sum()) == 0 and int((codes_buf[:, 16 + x.shape[1]:] != 3).sum()) == 0


SHAPES = [(1, 128, 128), (1, 1, 1), (1, 16, 16), (2, 130, 100), (7, 2048, 2048), (8, 100, 127), (9, 257, 129), (16, 640, 1000),
          (17, 2050, 2048), (31, 300, 4100), (33, 128, 64), (64, 2048, 512), (65, 129, 8192), (100, 1000, 144), (128, 256, 256),
          (129, 257, 384), (200, 2048, 2048), (300, 511, 1030), (520, 768, 640), (1, 40000, 256), (16, 128, 16384), (1000, 24, 256),
          (1, 25000, 1010), (5, 40000, 700), (13, 3001, 8400), (16, 130, 200000), (2, 12700, 2048), (32, 300, 1000), (24, 20000, 130), (9, 6144, 4097)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, dtype):
    w, sw = quantized(rows(n, k, torch.bfloat16, 1, wide=False), 128)
    sw = sw * (1 + 0.7 * torch.rand(sw.shape, device="cuda"))            # scales as checkpoints hold them: no powers of two
    xb = rows(m, k, torch.bfloat16, 2)
    x, sx = quantized(xb)
    want, mag = expect(x, sx, w, sw)
    out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    kernels.gemm_fp8(x, w, sw, out, sx)
    check_product(out, want, mag, k)
    whole = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    kernels.gemm_fp8(xb, w, sw, whole)                                    # quantised on the way: the same numbers
    check_product(whole, want, mag, k)
    again = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    kernels.gemm_fp8(xb, w, sw, again)
    assert torch.equal(whole, again)


@pytest.mark.parametrize("m", [1, 5, 20, 150])
def test_product_of_float32_rows_and_column_slices(m):
    n, k = 200, 320
    w, sw = quantized(rows(n, k, torch.float32, 1, wide=False), 128)
    big = rows(m, 1000, torch.float32, 2)
    for x in (big[:, 3:3 + k], big[:, 8:8 + k], big[:, 1:1 + k].to(torch.bfloat16)):
        xc, sx = quantized(x)
        want, mag = expect(xc, sx, w, sw)
        buf = torch.full((m + 2, 640), 7.0, dtype=torch.bfloat16, device="cuda")
        out = buf[1:-1, 5:5 + n]
        kernels.gemm_fp8(x, w, sw, out)
        check_product(out, want, mag, k)
        buf[1:-1, 5:5 + n] = 7.0
        assert bool((buf == 7.0).all())                                   # nothing beside the result
        # codes and scales as column slices of larger tables, and a weight whose rows lie far apart
        cb = torch.zeros(m, 1024, dtype=torch.uint8, device="cuda").view(FP8)
        cb[:, 32:32 + k] = xc
        wide = torch.zeros(n, 2048, dtype=torch.uint8, device="cuda").view(FP8)
        wide[:, 64:64 + k] = w
        st = torch.empty(sx.shape[1], m, device="cuda")
        st.t().copy_(sx)
        kernels.gemm_fp8(cb[:, 32:32 + k], wide[:, 64:64 + k], sw, out, st.t())
        check_product(out, want, mag, k)


@pytest.mark.parametrize("m", [1, 12, 40, 140])
def test_what_is_behind_the_columns_is_not_read(m):
    """Codes that follow a row's last column, in the padding or in the next columns, are NaN."""
    n, k = 130, 200
    nan = torch.full((max(m, n), 512), 0x7F, dtype=torch.uint8, device="cuda")
    wb, xb = nan[:n].clone().view(FP8), nan[:m].clone().view(FP8)
    w, x = wb[:, 16:16 + k], xb[:, 16:16 + k]
    wc, sw = quantized(rows(n, k, torch.bfloat16, 1, wide=False), 128)
    xc, sx = quantized(rows(m, k, torch.bfloat16, 2))
    w.copy_(wc)
    x.copy_(xc)
    out = torch.empty(m, n, device="cuda")
    kernels.gemm_fp8(x, w, sw, out, sx)
    want, mag = expect(xc, sx, wc, sw)
    check_product(out, want, mag, k)


@pytest.mark.parametrize("m", [3, 40, 140])
def test_a_number_that_is_none_stays_in_its_row(m):
    n, k = 256, 512
    w, sw = quantized(rows(n, k, torch.bfloat16, 1, wide=False), 128)
    x = rows(m, k, torch.bfloat16, 2)
    clean = torch.empty(m, n, device="cuda")
    kernels.gemm_fp8(x, w, sw, clean)
    x[1, 300] = float("nan")
    x[2, 3] = float("inf")
    out = torch.empty(m, n, device="cuda")
    kernels.gemm_fp8(x, w, sw, out)
    assert bool(torch.isnan(out[1:3]).all())
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(out[keep], clean[keep])


def test_offsets_beyond_32_bits():
    """A weight and rows of more than 2^32 codes: the last rows are what they are alone."""
    n, k = 540_000, 8192
    w = torch.zeros(n, k, dtype=torch.uint8, device="cuda").view(FP8)
    sw = torch.ones(-(-n // 128), 64, device="cuda")
    tail, st = quantized(rows(300, k, torch.bfloat16, 1, wide=False), 128)
    first = n - 300 - (n - 300) % 128                                     # a block of scales starts there
    w[first:first + 300].copy_(tail)
    sw[first // 128:first // 128 + 3] = st
    for m in (3, 20, 40, 200):
        x = rows(m, k, torch.bfloat16, m)
        out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
        kernels.gemm_fp8(x, w, sw, out)
        xc, sx = quantized(x)
        want, mag = expect(xc, sx, tail, st)
        check_product(out[:, first:first + 300], want, mag, k)
        assert bool((out[:, :first] == 0).all()) and bool((out[:, first + 300:] == 0).all())
    del w, out
    x = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    x[-5:] = rows(5, k, torch.bfloat16, 9)
    codes, scales = kernels.fp8_empty(n, k, "cuda"), torch.empty(n, 64, device="cuda")
    kernels.fp8_quantize_rows(x, codes, scales)
    want, ws = codes_of(x[-5:])
    assert same(codes[-5:], want) and torch.equal(scales[-5:].double(), ws) and bool((scales[:-5] == 1).all())
    kernels.fp8_quantize_blocks(x, codes, scales := torch.empty(-(-n // 128), 64, device="cuda"))
    want, ws = codes_of(x[n - n % 128 if n % 128 else n - 128:], 128)
    assert same(codes[n - want.shape[0]:], want) and torch.equal(scales[-1:].double(), ws)


def test_out_shares_no_memory_with_an_operand():
    k = 256
    w, sw = quantized(rows(256, k, torch.bfloat16, 1, wide=False), 128)
    x = rows(20, k, torch.bfloat16, 2)
    with pytest.raises(kernels.KernelError, match="shares memory"):
        kernels.gemm_fp8(x, w, sw, x)
    with pytest.raises(kernels.KernelError, match="shares memory"):
        kernels.gemm_fp8(x, w, sw, w.view(torch.bfloat16).view(-1)[:20 * 256].view(20, 256))
    buf = torch.empty(20, 600, dtype=torch.bfloat16, device="cuda")       # side by side is no overlap
    buf[:, :k] = x
    kernels.gemm_fp8(buf[:, :k], w, sw, buf[:, 300:556])
    want, mag = expect(*quantized(x), w, sw)
    check_product(buf[:, 300:556], want, mag, k)
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    with pytest.raises(kernels.KernelError, match="scratch holds"):
        kernels.gemm_fp8(x, w, sw, torch.empty(20, 256, device="cuda"), scratch=small)


def test_scratch_lies_apart():
    k = 256
    w, sw = quantized(rows(256, k, torch.bfloat16, 1, wide=False), 128)
    out = torch.empty(20, 256, device="cuda")
    buf = torch.empty(64 << 10, dtype=torch.uint8, device="cuda")
    x = buf[:20 * k * 2].view(torch.bfloat16).view(20, k)
    x.copy_(rows(20, k, torch.bfloat16, 2))
    bytes_ = kernels.gemm_fp8_scratch_bytes(x)
    for scratch in (buf[:bytes_], buf[20 * k * 2 - 16:], out.view(torch.uint8).view(-1), w.view(torch.uint8).view(-1)):
        with pytest.raises(kernels.KernelError, match="scratch shares memory"):
            kernels.gemm_fp8(x, w, sw, out, scratch=scratch)
    kernels.gemm_fp8(x, w, sw, out, scratch=buf[20 * k * 2:20 * k * 2 + bytes_])
    check_product(out, *expect(*quantized(x), w, sw), k)


FIRST = """
import torch
from inf_engine_b200 import kernels
M, N, K = {m}, {n}, {k}
w = torch.ones(N, K, device="cuda")
codes, scales = kernels.fp8_empty(N, K, "cuda"), torch.empty(-(-N // 128), -(-K // 128), device="cuda")
x, out = torch.ones(M, K, device="cuda", dtype=torch.bfloat16), torch.zeros(M, N, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    kernels.fp8_quantize_blocks(w, codes, scales)
    kernels.gemm_fp8(x, codes, scales, out)
g.replay()
torch.cuda.synchronize()
assert bool((out == K).all())
assert kernels.gemm_fp8_error() == 0
"""


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (12, 256, 512), (16, 13000, 2048), (24, 256, 1024), (100, 256, 1024), (300, 5120, 512)])
def test_the_first_call_of_a_program_may_be_captured(m, n, k):
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST.format(m=m, n=n, k=k)], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0, r.stderr[-1500:]


def test_empty_products():
    w, sw = quantized(rows(20, 64, torch.bfloat16), 128)
    kernels.gemm_fp8(torch.empty(0, 64, device="cuda"), w, sw, torch.empty(0, 20, device="cuda"))
    kernels.fp8_quantize_rows(torch.empty(0, 64, device="cuda"), kernels.fp8_empty(0, 64, "cuda"), torch.empty(0, 1, device="cuda"))


@pytest.mark.parametrize("m", [4, 40, 200])
def test_captured_and_on_another_stream(m):
    n, k = 384, 640
    w, sw = quantized(rows(n, k, torch.bfloat16, 1, wide=False), 128)
    x = rows(m, k, torch.bfloat16, 2)
    out = torch.empty(m, n, device="cuda")
    kernels.gemm_fp8(x, w, sw, out)
    other, third = rows(m, k, torch.bfloat16, 3), rows(m, k, torch.bfloat16, 4)
    want = []
    for y in (other, third):
        kernels.gemm_fp8(y, w, sw, out)
        want.append(out.clone())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph, second, out2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.empty(m, n, device="cuda")
    with torch.cuda.graph(graph, stream=side):
        kernels.gemm_fp8(x, w, sw, out)
    with torch.cuda.graph(second, stream=side):
        kernels.gemm_fp8(third, w, sw, out2)
    for _ in range(3):
        x.copy_(other)
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(out2, want[1])
    # two products at once on two streams
    a, b = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s1):
            kernels.gemm_fp8(other, w, sw, a)
        with torch.cuda.stream(s2):
            kernels.gemm_fp8(third, w, sw, b)
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])

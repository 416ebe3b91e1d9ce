"""The operators around a served model's matrix products and its next token: quantising rows and weights to 8 bits, the
product of the two, the history of a request's tokens, and the logits adjusted by it, by biases and by masks.

``run`` computes a case in elementary torch operations, or, where ``own`` is set, through this package's kernels.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 128          # columns that share a scale
TOP = 448.0          # the largest e4m3 number


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # the rows of a decode step of a small batch on their way into a projection
        {"name": "rows 7x2048", "op": "rows", "m": 7, "k": 2048, "dtype": "bfloat16"},
        # the widest activations of a whole step's prompt tokens
        {"name": "rows 4096x8192", "op": "rows", "m": 4096, "k": 8192, "dtype": "bfloat16"},
        # a stacked gate/up weight at load
        {"name": "blocks 16384x2048", "op": "blocks", "m": 16384, "k": 2048, "dtype": "bfloat16"},
        # a 32-bit weight whose sides are no multiples of a block
        {"name": "blocks 1000x2040 f32", "op": "blocks", "m": 1000, "k": 2040, "dtype": "float32"},
        # one request's output projection in a decode step: latency
        {"name": "product 1x2048x2048", "op": "product", "m": 1, "n": 2048, "k": 2048, "out": "bfloat16"},
        # the head over a decode batch: the largest weight that is streamed
        {"name": "product 6x128256x2048 f32", "op": "product", "m": 6, "n": 128256, "k": 2048, "out": "float32"},
        # a step of a batch of decode tokens beside a short prompt portion
        {"name": "product 77x2048x8192", "op": "product", "m": 77, "n": 2048, "k": 8192, "out": "bfloat16"},
        # prompts: the tensor cores' rate
        {"name": "product 4096x8192x8192", "op": "product", "m": 4096, "n": 8192, "k": 8192, "out": "bfloat16"},
        # a few requests with penalties over what they said, a small vocabulary
        {"name": "adjust 3x32000", "op": "adjust", "m": 3, "v": 32000, "dtype": "float32", "penalties": True, "said": 300,
         "biases": 0, "masks": 0, "allowed": 1.0},
        # a full batch with everything: long histories, biases, every other row held to a grammar
        {"name": "adjust 64x128256 all", "op": "adjust", "m": 64, "v": 128256, "dtype": "float32", "penalties": True, "said": 4000,
         "biases": 100, "masks": 32, "allowed": 0.02},
        # the tokens of one decode step go into their requests' histories
        {"name": "append 64x1", "op": "history", "slots": 64, "requests": 64, "tokens": 1, "prompt": 0, "v": 128256, "fresh": False},
        # requests that enter (or come back) with everything they hold
        {"name": "enter 64x4096", "op": "history", "slots": 64, "requests": 64, "tokens": 4096, "prompt": 3000, "v": 128256,
         "fresh": True},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "blocks", "product", "product", "adjust", "adjust", "history"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "rows":
        return {"op": op, "m": _spread(rng, 1, 4000), "k": _spread(rng, 50, 8000), "dtype": dtype}
    if op == "blocks":
        return {"op": op, "m": _spread(rng, 30, 8000), "k": _spread(rng, 50, 4000), "dtype": dtype}
    if op == "product":
        # few rows as often as many; widths of projections, odd ones among them
        m = rng.choice([_spread(rng, 1, 20), _spread(rng, 1, 4000)])
        k = _spread(rng, 100, 8000)
        return {"op": op, "m": m, "n": _spread(rng, 100, 16000), "k": k if rng.random() < 0.3 else -(-k // 64) * 64,
                "out": rng.choice(["bfloat16", "bfloat16", "float32"])}
    if op == "adjust":
        penalties = rng.random() < 0.7
        masks = not penalties or rng.random() < 0.4
        m = _spread(rng, 1, 60)
        return {"op": op, "m": m, "v": _spread(rng, 1000, 128000), "dtype": dtype, "penalties": penalties,
                "said": _spread(rng, 1, 4000), "biases": rng.choice([0, 0, _spread(rng, 1, 100)]),
                "masks": rng.randint(1, m) if masks else 0, "allowed": rng.choice([0.001, 0.02, 0.3, 0.9])}
    requests = rng.randint(1, 64)
    tokens = rng.choice([1, _spread(rng, 1, 4000)])
    return {"op": op, "slots": rng.randint(requests, 64), "requests": requests, "tokens": tokens, "prompt": rng.randint(0, tokens),
            "v": _spread(rng, 1000, 128000), "fresh": rng.random() < 0.5}


# ---------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _activations(g, m, k, dtype):
    """Rows as a norm leaves them: a scale of its own for every column, a few columns far larger than the others."""
    x = torch.randn(m, k, generator=g, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    x *= torch.where(torch.rand(k, generator=g, device=DEVICE) < 0.004, 30.0, 1.0)
    return x.to(dtype)


def _weight_codes(g, n, k):
    """A weight as a checkpoint stores it: e4m3 codes, and for each 128 x 128 block the scale largest / 448, which is no power
    of two.  Rows lie 16-byte multiples apart, as every projection's do."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    pitch = -(-k // 16) * 16
    codes = torch.zeros(n, pitch, dtype=torch.float8_e4m3fn, device=DEVICE)[:, :k]
    scales = torch.empty(nb, kb, device=DEVICE)
    step = 64 * BLOCK
    for r in range(0, n, step):
        rows = min(step, n - r)
        w = torch.zeros(-(-rows // BLOCK) * BLOCK, kb * BLOCK, device=DEVICE)
        w[:rows, :k] = 0.02 * torch.randn(rows, k, generator=g, device=DEVICE)
        w = w.view(-1, BLOCK, kb, BLOCK)
        s = w.abs().amax(dim=(1, 3)).clamp_min(1e-8) / TOP
        scales[r // BLOCK:r // BLOCK + s.shape[0]] = s
        codes[r:r + rows] = (w / s[:, None, :, None]).view(-1, kb * BLOCK)[:rows, :k].to(torch.float8_e4m3fn)
    return codes, scales


def _tokens(g, shape, v):
    """Token ids as text has them: a few very often, most hardly ever."""
    u = torch.rand(shape, generator=g, device=DEVICE)
    return (torch.exp(u * math.log(v)) - 1).long().clamp_(0, v - 1).to(torch.int32)


def _words(v):
    return -(-v // 32)


def _pack(bits):
    """bool [rows, v] -> int32 [rows, words], bit t % 32 of word t / 32."""
    rows, v = bits.shape
    padded = torch.zeros(rows, _words(v) * 32, dtype=torch.int64, device=bits.device)
    padded[:, :v] = bits
    at = torch.arange(32, device=bits.device)
    return (padded.view(rows, -1, 32) << at).sum(-1).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op in ("rows", "blocks"):
        m, k = case["m"], case["k"]
        dtype = getattr(torch, case["dtype"])
        x = _activations(g, m, k, dtype) if op == "rows" else (0.02 * torch.randn(m, k, generator=g, device=DEVICE)).to(dtype)
        groups = m if op == "rows" else -(-m // BLOCK)
        return {"op": op, "x": x, "codes": torch.zeros(m, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=DEVICE)[:, :k],
                "scales": torch.zeros(groups, -(-k // BLOCK), device=DEVICE)}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        codes, scales = _weight_codes(g, n, k)
        return {"op": op, "x": _activations(g, m, k, torch.bfloat16), "w": codes, "w_scales": scales,
                "out": torch.empty(m, n, dtype=getattr(torch, case["out"]), device=DEVICE)}
    if op == "adjust":
        m, v = case["m"], case["v"]
        s = {"op": op, "logits": (3.0 * torch.randn(m, v, generator=g, device=DEVICE)).to(getattr(torch, case["dtype"])),
             "out": torch.empty(m, v, device=DEVICE)}
        for name in ("slots", "penalties", "counts", "seen", "bias_start", "bias_ids", "bias_values", "mask_rows", "masks"):
            s[name] = None
        if case["penalties"]:
            n_slots = m + 2
            said, read = _tokens(g, (n_slots, case["said"]), v).long(), _tokens(g, (n_slots, case["said"]), v).long()
            s["counts"] = torch.zeros(n_slots, v, dtype=torch.int32, device=DEVICE)
            s["counts"].scatter_add_(1, said, torch.ones_like(said, dtype=torch.int32))
            bits = s["counts"] > 0
            bits.scatter_(1, read, True)
            s["seen"] = _pack(bits)
            s["slots"] = torch.randperm(n_slots, generator=g, device=DEVICE)[:m].to(torch.int32)
            # the factor for repetition, what is taken off once, what is taken off for each time
            s["penalties"] = torch.rand(m, 3, generator=g, device=DEVICE) * torch.tensor([0.4, 0.8, 0.5], device=DEVICE)
            s["penalties"] += torch.tensor([1.0, 0.0, 0.0], device=DEVICE)
        if case["biases"]:
            b = case["biases"]
            s["bias_start"] = (torch.arange(m + 1, device=DEVICE) * b).to(torch.int32)
            s["bias_ids"] = torch.randint(0, v, (m * b,), generator=g, device=DEVICE, dtype=torch.int32)
            s["bias_values"] = 4.0 * torch.randn(m * b, generator=g, device=DEVICE)
        if case["masks"]:
            s["masks"] = _pack(torch.rand(case["masks"], v, generator=g, device=DEVICE) < case["allowed"])
            rows = torch.full((m,), -1, dtype=torch.int32, device=DEVICE)
            rows[torch.randperm(m, generator=g, device=DEVICE)[:case["masks"]]] = torch.arange(
                case["masks"], dtype=torch.int32, device=DEVICE)
            s["mask_rows"] = rows
        return s
    n_slots, r, t, v = case["slots"], case["requests"], case["tokens"], case["v"]
    lengths = torch.randint(max(1, t // 2), t + 1, (r,), generator=g, device=DEVICE)
    starts = torch.zeros(r + 1, dtype=torch.int32, device=DEVICE)
    starts[1:] = lengths.cumsum(0)
    old = _tokens(g, (n_slots, 200), v).long()
    counts = torch.zeros(n_slots, v, dtype=torch.int32, device=DEVICE)
    counts.scatter_add_(1, old, torch.ones_like(old, dtype=torch.int32))
    return {"op": op, "fresh": case["fresh"], "counts": counts, "seen": _pack(counts > 0),
            "slots": torch.randperm(n_slots, generator=g, device=DEVICE)[:r].to(torch.int32), "starts": starts,
            "tokens": _tokens(g, (int(lengths.sum()),), v),
            "n_prompt": torch.clamp(lengths, max=case["prompt"]).to(torch.int32)}


# ---------------------------------------------------------------------------- the plain form
def _scale_of(largest):
    """2^ceil(log2(largest / 448)): the fraction of a float in [0.5, 1) says on which side of a power of two it lies."""
    fraction, exponent = torch.frexp(largest)
    exponent = exponent - 9 + (fraction > TOP / 512.0)
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), exponent.clamp_min(-126)), 1.0)


def _padded(x, rows, cols):
    out = torch.zeros(rows, cols, device=x.device)
    out[:x.shape[0], :x.shape[1]] = x
    return out


def _quantize(x, high):
    """Codes and scales of groups of ``high`` rows x 128 columns."""
    m, k = x.shape
    mb, kb = -(-m // high), -(-k // BLOCK)
    p = _padded(x, mb * high, kb * BLOCK).view(mb, high, kb, BLOCK)
    scales = _scale_of(p.abs().amax(dim=(1, 3)))
    codes = (p / scales[:, None, :, None]).view(mb * high, kb * BLOCK)[:m, :k].to(torch.float8_e4m3fn)
    return codes, scales


def _values(codes, scales, high):
    """The numbers that codes and scales stand for, float32."""
    m, k = codes.shape
    s = scales.repeat_interleave(high, 0)[:m] if high > 1 else scales
    return codes.float() * s.repeat_interleave(BLOCK, 1)[:, :k]


def _unpacked(words, v):
    at = torch.arange(32, dtype=torch.int32, device=words.device)
    return ((words[:, :, None] >> at) & 1).view(words.shape[0], -1)[:, :v].bool()


def _plain_adjust(s):
    x = s["logits"].float()
    m, v = x.shape
    if s["penalties"] is not None:
        slots, held = s["slots"].long().clamp_min(0), (s["slots"] >= 0)[:, None]
        factor, once, each = s["penalties"][:, 0:1], s["penalties"][:, 1:2], s["penalties"][:, 2:3]
        seen = _unpacked(s["seen"][slots], v) & held
        counts = s["counts"][slots] * held
        x = torch.where(seen, torch.where(x < 0, x * factor, x / factor), x)
        x = torch.where(counts > 0, x - (each * counts + once), x)
    if s["bias_ids"] is not None:
        rows = torch.searchsorted(s["bias_start"], torch.arange(s["bias_ids"].shape[0], device=x.device), right=True) - 1
        x = x.index_put((rows, s["bias_ids"].long()), s["bias_values"], accumulate=True)
    if s["masks"] is not None:
        allowed = _unpacked(s["masks"][s["mask_rows"].long().clamp_min(0)], v)
        x = torch.where(allowed | (s["mask_rows"] < 0)[:, None], x, -math.inf)
    return x


def _plain_history(s):
    counts, seen = s["counts"], s["seen"]
    v, words = counts.shape[1], seen.shape[1]
    slots = s["slots"].long()
    if s["fresh"]:
        counts[slots] = 0
        seen[slots] = 0
    starts = s["starts"].long()
    n = s["tokens"].shape[0]
    of = torch.searchsorted(starts, torch.arange(n, device=starts.device), right=True) - 1      # whose token it is
    generated = torch.arange(n, device=starts.device) - starts[of] >= s["n_prompt"].long()[of]
    at = slots[of] * v + s["tokens"].long()
    counts.view(-1).index_add_(0, at, generated.to(torch.int32))
    each = torch.unique(at)
    word, bit = each // v * words + each % v // 32, (each % v % 32).to(torch.int32)
    flat = seen.view(-1)
    new = ((flat[word] >> bit) & 1) == 0
    flat.index_add_(0, word, torch.where(new, torch.ones_like(bit) << bit, 0))
    return counts, seen


def _plain(s):
    op = s["op"]
    if op in ("rows", "blocks"):
        codes, scales = _quantize(s["x"].float(), 1 if op == "rows" else BLOCK)
        return {"codes": codes, "scales": scales}
    if op == "product":
        x = _values(*_quantize(s["x"].float(), 1), 1)
        return (x @ _values(s["w"], s["w_scales"], BLOCK).t()).to(s["out"].dtype)
    if op == "adjust":
        return _plain_adjust(s)
    counts, seen = _plain_history(s)
    return {"counts": counts, "seen": seen}


# ---------------------------------------------------------------------------- one pass
def run(state):
    if not own:
        return _plain(state)
    from inf_engine_b200 import kernels

    s, op = state, state["op"]
    if op == "rows":
        kernels.fp8_quantize_rows(s["x"], s["codes"], s["scales"])
        return {"codes": s["codes"], "scales": s["scales"]}
    if op == "blocks":
        kernels.fp8_quantize_blocks(s["x"], s["codes"], s["scales"])
        return {"codes": s["codes"], "scales": s["scales"]}
    if op == "product":
        kernels.gemm_fp8(s["x"], s["w"], s["w_scales"], s["out"])
        return s["out"]
    if op == "adjust":
        kernels.adjust_logits(s["logits"], s["out"], s["slots"], s["penalties"], s["counts"], s["seen"], s["bias_start"],
                              s["bias_ids"], s["bias_values"], s["mask_rows"], s["masks"])
        return s["out"]
    if s["fresh"]:
        kernels.history_reset(s["counts"], s["seen"], s["slots"])
    kernels.history_append(s["counts"], s["seen"], s["tokens"], s["slots"], s["starts"], s["n_prompt"])
    return {"counts": s["counts"], "seen": s["seen"]}


def work(case):
    op = case["op"]
    if op in ("rows", "blocks"):
        m, k = case["m"], case["k"]
        groups = (m if op == "rows" else -(-m // BLOCK)) * -(-k // BLOCK)
        return {"bytes": m * k * ((2 if case["dtype"] == "bfloat16" else 4) + 1) + 4 * groups, "flops": 2 * m * k}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": 2 * m * k + n * k + 4 * kb * -(-n // BLOCK) + m * n * (2 if case["out"] == "bfloat16" else 4),
                "flops": 2 * m * n * k}
    if op == "adjust":
        m, v = case["m"], case["v"]
        b = m * v * ((2 if case["dtype"] == "bfloat16" else 4) + 4) + 8 * m * case["biases"] + 4 * case["masks"] * _words(v)
        if case["penalties"]:
            b += m * (4 * _words(v) + 4 * min(v, 2 * case["said"]) + 16)
        return {"bytes": b, "flops": 2 * m * v}
    tokens = case["requests"] * max(1, 3 * case["tokens"] // 4)
    b = tokens * (4 + 16) + 12 * case["requests"]
    if case["fresh"]:
        b += case["requests"] * (4 * case["v"] + 4 * _words(case["v"]))
    return {"bytes": b, "flops": 2 * tokens}


# ---------------------------------------------------------------------------- the definition in 64 bits
def _exact_codes(x, high):
    """The nearest e4m3 numbers (ties to even) of float64 x over its groups' scales, and the scales."""
    m, k = x.shape
    mb, kb = -(-m // high), -(-k // BLOCK)
    p = torch.zeros(mb * high, kb * BLOCK, dtype=torch.float64, device=x.device)
    p[:m, :k] = x
    p = p.view(mb, high, kb, BLOCK)
    top = p.abs().amax(dim=(1, 3))
    scale = torch.ones_like(top)
    exponent = torch.floor(torch.log2(top.clamp_min(1e-300) / TOP)) - 1      # certainly too small: one or two steps up
    for _ in range(3):
        exponent = torch.where(top > TOP * torch.exp2(exponent), exponent + 1, exponent)
    scale = torch.where(top > 0, torch.exp2(exponent.clamp_min(-126)), scale)
    q = p / scale[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.round(q / step) * step
    return q.view(mb * high, kb * BLOCK)[:m, :k], scale


def exact(case, seed):
    op = case["op"]
    if op == "history":
        return None                    # whole numbers
    s = prepare(case, seed)
    if op in ("rows", "blocks"):
        codes, scales = _exact_codes(s["x"].double(), 1 if op == "rows" else BLOCK)
        return {"codes": codes, "scales": scales}
    if op == "product":
        codes, scales = _exact_codes(s["x"].double(), 1)
        k, n = case["k"], case["n"]
        out = torch.zeros(case["m"], n, dtype=torch.float64, device=DEVICE)
        for r in range(0, n, 64 * BLOCK):                # slices of the weight, or 64 bits of all of it fill the card
            w = s["w"][r:r + 64 * BLOCK].double()
            ws = s["w_scales"].double()[r // BLOCK:r // BLOCK + 64]
            at = torch.arange(w.shape[0], device=DEVICE) // BLOCK
            cols = torch.arange(k, device=DEVICE) // BLOCK
            out[:, r:r + w.shape[0]] = (codes * scales[:, cols]) @ (w * ws[at][:, cols]).t()
        return out
    x = s["logits"].double().cpu().numpy()
    m, v = x.shape
    host = {name: t.cpu().numpy() for name, t in s.items() if isinstance(t, torch.Tensor)}
    for row in range(m):
        if "penalties" in host and host["slots"][row] >= 0:
            slot = host["slots"][row]
            factor, once, each = host["penalties"][row].astype(np.float64)
            at = np.nonzero(np.unpackbits(host["seen"][slot].view(np.uint8), bitorder="little")[:v])[0]
            x[row, at] = np.where(x[row, at] < 0, x[row, at] * factor, x[row, at] / factor)
            at = np.nonzero(host["counts"][slot])[0]
            x[row, at] -= each * host["counts"][slot][at] + once
        if "bias_ids" in host:
            at = slice(host["bias_start"][row], host["bias_start"][row + 1])
            np.add.at(x[row], host["bias_ids"][at], host["bias_values"][at].astype(np.float64))
        if "masks" in host and host["mask_rows"][row] >= 0:
            allowed = np.unpackbits(host["masks"][host["mask_rows"][row]].view(np.uint8), bitorder="little")[:v]
            x[row, allowed == 0] = -np.inf
    return torch.from_numpy(x)

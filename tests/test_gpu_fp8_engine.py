"""Models whose layers' matrices are kept in 8-bit floating point, through the engine.

The plain implementation runs with the numbers that the codes stand for and quantises the rows of every such product, in float32.  The
engine's bfloat16 activations differ from the plain ones, so near a border between two codes it takes the other, and the more the two
have drifted apart the less the two roundings have to do with each other.  Were they unrelated, each rounding would be off by a root
mean square of 2^-3 / m / sqrt(12) of a number with fraction m, 0.0255 over fractions spread evenly over [1, 2) (the mean of 1 / m^2 is
1/2), and the rows of a product would differ by sqrt(2) times that, 0.036.  Two layers hold eight products, whose errors are
independent and add as squares, with BF16_ROW_MAX for the rest: sqrt(8 * 0.036^2 + 0.02^2) = 0.104, a mean square over rows, and compared
with one.  That says that every part of a model meets the right matrix; how exact a product is, is tested on its own."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

import plain_llama
from helpers import TINY, make_model_dir, plain_inputs, random_tokens

pytestmark = pytest.mark.gpu
ROW_RMS = 0.104


def fake_quantized(x, high):
    from test_gpu_fp8 import codes_of
    codes, scales = codes_of(x, high)
    m, k = x.shape
    return (codes * scales.repeat_interleave(high, 0)[:m].repeat_interleave(128, 1)[:, :k]).float()


class Quantized:
    """Stands for a weight in ``h @ w.T``: the product of quantised rows and quantised blocks."""

    def __init__(self, w):
        self.w, self.T = w, self

    def float(self):
        return self

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        h, w = args
        return fake_quantized(h, 1) @ w.w.t()


def quantized_weights(weights, config):
    """The layers' matrices as the engine keeps them: stacked as it stacks them, then in blocks of 128 x 128."""
    out = dict(weights)
    for i in range(config["num_hidden_layers"]):
        p = f"model.layers.{i}."
        q, k, v = (weights[p + f"self_attn.{n}_proj.weight"] for n in "qkv")
        parts = fake_quantized(torch.cat([q, k, v]), 128).split([q.shape[0], k.shape[0], v.shape[0]])
        for n, w in zip("qkv", parts):
            out[p + f"self_attn.{n}_proj.weight"] = Quantized(w)
        gate, up = weights[p + "mlp.gate_proj.weight"], weights[p + "mlp.up_proj.weight"]
        both = fake_quantized(torch.stack([gate, up], 1).reshape(-1, gate.shape[1]), 128).view(-1, 2, gate.shape[1])
        out[p + "mlp.gate_proj.weight"], out[p + "mlp.up_proj.weight"] = Quantized(both[:, 0]), Quantized(both[:, 1])
        for n in ("self_attn.o_proj", "mlp.down_proj"):
            out[p + n + ".weight"] = Quantized(fake_quantized(weights[p + n + ".weight"], 128))
    return out


@pytest.mark.parametrize("name", ["tiny_d", "tiny_f", "tiny_e"])
def test_logits(tmp_path, name):
    from inf_engine_b200 import ModelRunner, StepEntry
    d = make_model_dir(tmp_path, name)
    config, weights = plain_inputs(d)
    toks = random_tokens(config["vocab_size"], 300, 11)
    ref = plain_llama.forward_logits(quantized_weights(weights, config), config, toks)
    r = ModelRunner.from_dir(d, dtype="bfloat16", page_size=16, n_pages=40, weights="fp8")
    r.open("x")
    rows = [r.step([StepEntry("x", toks[:270], list(range(270)))]).cpu().clone()]          # tiles
    rows.append(r.step([StepEntry("x", toks[270:282], list(range(12)))]).cpu().clone())    # twelve rows
    for t in toks[282:]:                                                                   # single tokens, replayed graphs
        rows.append(r.step([StepEntry("x", [t], [0])]).cpu().clone())
    got = torch.cat(rows)
    err = (got - ref).norm(dim=1) / ref.norm(dim=1)
    rms = float(err.square().mean().sqrt())
    assert rms <= ROW_RMS, rms
    from inf_engine_b200 import kernels
    kernels.check_device_errors()


def test_what_is_kept_in_eight_bits(tmp_path):
    from inf_engine_b200 import Engine, ModelRunner
    d = make_model_dir(tmp_path, "tiny_f")
    r = ModelRunner.from_dir(d, dtype="bfloat16", n_pages=8, weights="fp8")
    layer = r.model.layers[0]
    for lin in (layer.mixer.qkv, layer.mixer.o, layer.feedforward.gate_up, layer.feedforward.down):
        assert lin.weight.dtype is torch.float8_e4m3fn and lin.scales is not None
    assert layer.mixer.o_weight is None and r.model.head.weight.dtype is torch.bfloat16
    with pytest.raises(ValueError, match="bfloat16"):
        Engine.from_dir(d, dtype="float32", weights="fp8")
    with pytest.raises(ValueError, match="fp8"):
        ModelRunner.from_dir(d, dtype="bfloat16", weights="int4")


@pytest.mark.parametrize("m", [1, 7, 12, 40, 300])
def test_a_layers_products_are_the_definition(tmp_path, m):
    from inf_engine_b200 import ModelRunner
    from test_gpu_fp8 import check_product, codes_of, expect, rows
    d = make_model_dir(tmp_path, "tiny_f")
    _, weights = plain_inputs(d)
    r = ModelRunner.from_dir(d, dtype="bfloat16", n_pages=8, weights="fp8")
    p = "model.layers.1."
    stacked = torch.cat([weights[p + f"self_attn.{n}_proj.weight"] for n in "qkv"])
    for lin, w in ((r.model.layers[1].mixer.qkv, stacked), (r.model.layers[1].feedforward.down, weights[p + "mlp.down_proj.weight"])):
        x = rows(m, w.shape[1], torch.bfloat16, m)
        out = torch.empty(m, w.shape[0], dtype=torch.bfloat16, device="cuda")
        lin(x, out)
        want, mag = expect(*codes_of(x), *(t.cuda() for t in codes_of(w, 128)))
        check_product(out, want, mag, w.shape[1])


@pytest.mark.parametrize("family", ["barerax", "kipezen", "fovunex", "gavatar", "nurilorn", "nurasun"])
def test_other_families_run(tmp_path, family):
    """Every family's steps run with 8-bit matrices: finite logits, near those of the model as it is (two to four layers, each product off by
    2^-4 / sqrt(3) twice: well within half of the norm), and the same from a prompt in one portion as in three."""
    import importlib
    from inf_engine_b200 import ModelRunner, StepEntry
    models = importlib.import_module(f"{family}_models")
    names = {"barerax": "brx_c", "kipezen": "kpz_c", "fovunex": "fvx_w", "gavatar": "gav_w", "nurilorn": "nur_t", "nurasun": "sun_t"}
    d = getattr(models, f"make_{family}_dir")(tmp_path, names[family])
    toks = random_tokens(200, 40, 3)
    got = {}
    for weights in (None, "fp8"):
        r = ModelRunner.from_dir(d, dtype="bfloat16", page_size=8, n_pages=40, max_requests=2, weights=weights)
        r.open("x")
        first = r.step([StepEntry("x", toks[:30], [29])]).cpu().clone()
        rest = [r.step([StepEntry("x", [t], [0])]).cpu().clone() for t in toks[30:]]
        got[weights] = torch.cat([first, *rest])
        assert bool(torch.isfinite(got[weights]).all())
    kept = got[None]
    assert float(((got["fp8"] - kept).norm(dim=1) / kept.norm(dim=1)).median()) < 0.5


def test_the_whole_path_from_eight_bits_to_a_constrained_token(tmp_path):
    """Rows -> codes -> product -> logits -> penalties, biases, mask -> token -> history, over several steps."""
    from inf_engine_b200 import kernels
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    m, k, v, slots = 5, 640, 5003, 7
    w = 0.05 * torch.randn(v, k, generator=g, device="cuda")
    codes = kernels.fp8_empty(v, k, "cuda")
    scales = torch.empty(-(-v // 128), -(-k // 128), device="cuda")
    kernels.fp8_quantize_blocks(w, codes, scales)
    wq = codes.double() * scales.double().repeat_interleave(128, 0)[:v].repeat_interleave(128, 1)[:, :k]
    counts = torch.zeros(slots, v, dtype=torch.int32, device="cuda")
    seen = torch.zeros(slots, -(-v // 32), dtype=torch.int32, device="cuda")
    at = torch.tensor([6, 0, 3, 2, 5], dtype=torch.int32, device="cuda")
    pen = torch.tensor([[1.5, 0.4, 0.2]] * m, device="cuda")
    bias = (torch.tensor([0, 0, 2, 2, 2, 3], dtype=torch.int32, device="cuda"), torch.tensor([7, 9, 11], dtype=torch.int32, device="cuda"),
            torch.tensor([3.0, -2.0, 8.0], device="cuda"))
    mask = torch.zeros(1, seen.shape[1], dtype=torch.int32, device="cuda")
    mask[0, 5:40] = -1
    rows = torch.tensor([-1, -1, 0, -1, -1], dtype=torch.int32, device="cuda")
    logits, tokens = torch.empty(m, v, device="cuda"), torch.empty(m, dtype=torch.int32, device="cuda")
    count = torch.zeros(slots, v, dtype=torch.float64)
    for step in range(6):
        x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
        kernels.gemm_fp8(x, codes, scales, logits)
        kernels.adjust_logits(logits, logits, at, pen, counts, seen, *bias, rows, mask)
        kernels.argmax(logits, tokens)
        kernels.history_append(counts, seen, tokens, at)
        y = (fake_quantized(x, 1).double() @ wq.t()).cpu()
        for i, slot in enumerate(at.tolist()):
            had = count[slot] > 0
            z = torch.where(had, torch.where(y[i] < 0, y[i] * 1.5, y[i] / 1.5), y[i])
            z = torch.where(had, z - 0.2 * count[slot] - 0.4, z)
            for b in range(int(bias[0][i]), int(bias[0][i + 1])):
                z[int(bias[1][b])] += float(bias[2][b])
            if i == 2:
                z[:160], z[1280:] = -torch.inf, -torch.inf
            t = int(tokens[i])
            assert float(z.max() - z[t]) <= 1e-4 * float(z.max().abs())
            count[slot, t] += 1
    assert torch.equal(counts.cpu().double(), count)


def test_command_line(tmp_path):
    d = make_model_dir(tmp_path, "tiny_f")
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, str(root / "bin" / "generate_llama"), "--model-dir", str(d), "--prompt-ids", "5,17,3", "--n", "6",
                        "--weights", "fp8", "--presence-penalty", "0.5", "--frequency-penalty", "0.2", "--logit-bias", "7:1e6"],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.strip() == "0: 7,7,7,7,7,7"

"""Every family's model with its matrices in 8 bits: which matrices are kept so, that nothing keeps them in bfloat16 beside, and that a
prompt gives the same logits in one portion as in three.

Two cuts of a prompt differ by the order of sums in attention and by bfloat16 roundings, and near a border between two codes one cut may take
the other code.  Were the two cuts' roundings unrelated, each product's rows would differ by sqrt(2) * 0.0255 = 0.036 of their norm (a root
mean square; 0.0255 is that of a rounding to e4m3 over fractions spread evenly); with P products between prompt and logits, and
BF16_ROW_MAX for the rest, sqrt(P * 0.036^2 + 0.02^2) bounds a mean square over rows."""

import dataclasses
import importlib

import pytest
import torch

from test_gpu_fp8 import codes_of
from helpers import BF16_ROW_MAX, make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
# family: model of the tests, how many of its matrices have a block of scales each way
MODELS = {"barerax": ("brx_c", 9), "kipezen": ("kpz_c", 8), "fovunex": ("fvx_w", 11), "gavatar": ("gav_w", 3), "nurilorn": ("nur_t", 6),
          "nurasun": ("sun_t", 12), "llama": ("tiny_f", 8)}


def model_dir(tmp_path, family):
    name = MODELS[family][0]
    if family == "llama":
        return make_model_dir(tmp_path, name)
    return getattr(importlib.import_module(f"{family}_models"), f"make_{family}_dir")(tmp_path, name)


def runner(d, weights):
    from inf_engine_b200 import ModelRunner
    return ModelRunner.from_dir(d, dtype="bfloat16", page_size=8, n_pages=40, max_requests=2, weights=weights)


def held(obj, seen, path=""):
    """Every product and tensor that an object of the model holds, with the way to it."""
    from inf_engine_b200.parts.linear import Linear
    if id(obj) in seen:
        return
    seen.add(id(obj))
    if isinstance(obj, (torch.Tensor, Linear)):
        yield path, obj
    if isinstance(obj, dict):
        inner = obj.items()
    elif isinstance(obj, (list, tuple)):
        inner = enumerate(obj)
    elif type(obj).__module__.startswith("inf_engine_b200.parts") and type(obj).__name__ != "Runtime":
        inner = vars(obj).items()
    else:
        return
    for name, value in list(inner):
        yield from held(value, seen, f"{path}.{name}")


def check_kept(obj):
    """How many products hold codes; none that could holds anything else, and no part keeps a matrix of such a product beside it."""
    from inf_engine_b200.parts.linear import Linear
    everything = list(held(obj, set()))
    products = [(p, x) for p, x in everything if isinstance(x, Linear)]
    coded = [x for _, x in products if x.scales is not None]
    assert all(x.weight.dtype is torch.float8_e4m3fn and x.scales.dtype is torch.float32 for x in coded)
    for p, x in products:
        assert x.scales is not None or x.name == "head" or min(x.out_features, x.in_features) < 128, p
    shapes = {(x.out_features, x.in_features) for x in coded}
    beside = [p for p, x in everything if isinstance(x, torch.Tensor) and x.dtype is torch.bfloat16 and tuple(x.shape) in shapes
              and not p.startswith((".embedding", ".head"))]
    assert not beside
    return len(coded)


@pytest.mark.parametrize("family", MODELS)
def test_matrices_are_kept_as_codes_alone(tmp_path, family):
    r = runner(model_dir(tmp_path, family), "fp8")
    assert check_kept(r.model) == MODELS[family][1]


@pytest.mark.parametrize("family", MODELS)
def test_a_prompt_in_one_portion_as_in_three(tmp_path, family):
    from inf_engine_b200 import StepEntry
    d = model_dir(tmp_path, family)
    toks = random_tokens(200, 47, 3)

    def logits(cuts, weights):
        r, out, at = runner(d, weights), [], 0
        r.open("x")
        for n in cuts:
            out.append(r.step([StepEntry("x", toks[at:at + n], list(range(n)))]).cpu().clone())
            at += n
        return torch.cat(out)

    def rms(a, b):
        return float(((a - b).norm(dim=1) / b.norm(dim=1)).square().mean().sqrt())
    one, three, kept = logits([47], "fp8"), logits([19, 1, 27], "fp8"), logits([47], None)
    assert rms(three, one) <= (MODELS[family][1] * 0.036 ** 2 + BF16_ROW_MAX ** 2) ** 0.5
    assert rms(one, kept) > 2 * rms(logits([19, 1, 27], None), kept) and not torch.equal(one, kept)      # the codes are what is multiplied


def test_mixers_inside_another_let_go_of_their_matrices(tmp_path):
    """A parallel mixer of which one branch has no output projection of the kind that can be joined: each branch keeps its own product."""
    from inf_engine_b200.config import ParallelMixerSpec
    from inf_engine_b200.config.spec import MinGRUSpec
    from inf_engine_b200.parts.registry import build_mixer, mixer_class
    from inf_engine_b200.parts.runtime import Runtime
    r = runner(model_dir(tmp_path, "llama"), None)
    spec = r.spec.layers[0].mixer
    other = MinGRUSpec(kind="mingru", hidden=spec.hidden, width=256, z_proj="z", z_bias="zb", x_proj="x", x_bias="xb", gate_proj="g", o_proj="o")
    both = ParallelMixerSpec(kind="parallel", hidden=spec.hidden, branches=(spec, other))
    tensors = {n: torch.randn(t.shape, device="cuda").to(torch.bfloat16) for n, t in mixer_class(both).expected_tensors(both).items()}
    mixer = build_mixer(both, tensors, Runtime("cuda:0", torch.bfloat16, "fp8"))
    assert not mixer.joint and check_kept(mixer) == 4
    joint = ParallelMixerSpec(kind="parallel", hidden=spec.hidden, branches=(spec, dataclasses.replace(spec, o_proj="o2")))
    tensors["o2"] = torch.randn(tensors[spec.o_proj].shape, device="cuda").to(torch.bfloat16)
    mixer = build_mixer(joint, tensors, Runtime("cuda:0", torch.bfloat16, "fp8"))
    assert mixer.joint and check_kept(mixer) == 3
    want = torch.cat([tensors[spec.o_proj], tensors["o2"]], dim=1)
    assert torch.equal(mixer.o.weight.float(), codes_of(want, 128)[0].float())

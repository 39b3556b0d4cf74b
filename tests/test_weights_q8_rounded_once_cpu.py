"""Matrices on their way to 8-bit codes and back are rounded once: from what is stored to codes, from stored codes to the engine's type."""
import warnings

import pytest
import torch

import q8_linear_refs as refs
from arle_b200.engine.loading import random_model
from arle_b200.parts.moe import RoutedExperts, RoutedExpertsSpec
from arle_b200.weights import random_tensors
from arle_b200.weights.q8 import StoredQ8
from test_weights_q8_engine_cpu import CONFIG, q8_kernels  # noqa: F401 (a fixture)

LAYER = "model.layers.0."


def _tensors(config, seed, kinds):
    """A model's tensors, its matrices by ``kinds(name, float32 matrix)``; and the model they are for."""
    model = random_model(config, seed, "float32", "cpu")
    out = {}
    for name, t in random_tensors(model.weight_decls(), seed, dtype=torch.float32).items():
        out[name] = kinds(name, t) if "_proj" in name else t
    return out, model


def _stored(t, seed=1):
    n, k = t.shape
    g = torch.Generator().manual_seed(seed)
    scales = t.abs().max() / 400.0 * (0.5 + torch.rand(-(-n // 128), -(-k // 128), generator=g))
    full = scales.repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]
    return StoredQ8((t / full).clamp(-448, 448).to(refs.E4M3), scales)


def _numbers(q):
    n, k = q.shape
    return refs.host(q.codes) * q.scales.double().repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes_of_matrices_stored_in_32_bits(q8_kernels, dtype):  # noqa: F811
    tensors, model = _tensors(dict(CONFIG, num_hidden_layers=1), 3, lambda name, t: t)
    model.load(tensors, dtype, "cpu", weight_dtype="float8_e4m3")
    mixer, ffn = model.blocks[0].mixer, model.blocks[0].ffn
    attn = [tensors[LAYER + f"self_attn.{r}_proj.weight"] for r in "qkvo"]
    mlp = [tensors[LAYER + f"mlp.{r}_proj.weight"] for r in ("gate", "up", "down")]
    for got, want in ((mixer.w_qkv, torch.cat(attn[:3])), (mixer.w_o, attn[3]), (ffn.w_down, mlp[2])):
        c, s = refs.quantize_weight(want.double())
        assert torch.equal(refs.host(got.codes), c) and torch.equal(got.scales.double(), s)
        twice, _ = refs.quantize_weight(want.bfloat16().double())
        assert not torch.equal(twice, c)                   # (the numbers tell the two apart)
    rows = refs.host(ffn.w_gate_up.codes).view(-1, 2, 128, ffn.w_gate_up.shape[1])
    for j in (0, 1):
        c, _ = refs.quantize_weight(mlp[j].double())
        assert torch.equal(rows[:, j].reshape(-1, rows.shape[3])[: c.shape[0]], c)


def test_stored_codes_that_end_inside_a_block_are_found_anew_from_their_own_numbers(q8_kernels):  # noqa: F811
    """Key and value matrices of 64 rows share a block: no scale of theirs fits it.  The codes are those of code * scale in float32, and the loader says so."""
    tensors, model = _tensors(dict(CONFIG, num_hidden_layers=1), 3, lambda name, t: _stored(t))
    with pytest.warns(UserWarning, match="k_proj"):
        model.load(tensors, torch.bfloat16, "cpu", weight_dtype="float8_e4m3")
    qkv = [tensors[LAYER + f"self_attn.{r}_proj.weight"] for r in "qkv"]
    c, s = refs.quantize_weight(torch.cat([_numbers(t).float() for t in qkv]).double())
    got = model.blocks[0].mixer.w_qkv
    assert torch.equal(refs.host(got.codes), c) and torch.equal(got.scales.double(), s)
    o = model.blocks[0].mixer.w_o                          # these keep their own
    assert torch.equal(o.scales, tensors[LAYER + "self_attn.o_proj.weight"].scales)


def test_nothing_is_said_where_codes_are_kept(q8_kernels):  # noqa: F811
    tensors, model = _tensors(dict(CONFIG, num_hidden_layers=1, head_dim=128), 3, lambda name, t: _stored(t))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        model.load(tensors, torch.bfloat16, "cpu", weight_dtype="float8_e4m3")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_stored_codes_in_the_engine_s_type(dtype):
    """Without ``weight_dtype`` stored codes become numbers of the engine's type, rounded to it once: a float32 engine has code * scale as float32 holds it."""
    tensors, model = _tensors(dict(CONFIG, num_hidden_layers=1, tie_word_embeddings=False), 3, lambda name, t: _stored(t))
    tensors["lm_head.weight"] = _stored(tensors["lm_head.weight"])
    model.load(tensors, dtype, "cpu")
    mixer, ffn = model.blocks[0].mixer, model.blocks[0].ffn
    want = {r: _numbers(tensors[LAYER + f"{p}.{r}_proj.weight"]).to(torch.float32).to(dtype)
            for p, rs in (("self_attn", "qkvo"), ("mlp", ("gate", "up", "down"))) for r in rs}
    assert torch.equal(mixer.w_qkv, torch.cat([want[r] for r in "qkv"])) and torch.equal(mixer.w_o, want["o"])
    assert torch.equal(ffn.w_gate_up[0::2], want["gate"]) and torch.equal(ffn.w_gate_up[1::2], want["up"]) and torch.equal(ffn.w_down, want["down"])
    assert torch.equal(model.head, _numbers(tensors["lm_head.weight"]).to(torch.float32).to(dtype))
    assert model.head.dtype == mixer.w_o.dtype == ffn.w_down.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gated", [True, False])
def test_stored_codes_of_experts(dtype, gated):
    """Parts that know nothing of codes load them like any other tensor, experts (which are stacked) among them."""
    spec = RoutedExpertsSpec(prefix="m.", hidden_size=130, num_experts=3, top=1, expert_ff=40, correction=False, gated=gated, activation="silu" if gated else "square_relu")
    loaded = []
    for stored in (True, False):
        part = RoutedExperts(spec)
        tensors = {}
        for i, d in enumerate(part.weight_decls()):
            q = _stored(torch.randn(d.shape, generator=torch.Generator().manual_seed(i)), i)
            tensors[d.name] = q if stored else q.to(dtype=dtype)
        part.load(tensors, dtype, "cpu")
        loaded.append(part)
    for name in ("w_router", "w_gate_up", "w_down"):
        a, b = (getattr(p, name) for p in loaded)
        assert a.dtype == b.dtype == dtype and torch.equal(a, b)

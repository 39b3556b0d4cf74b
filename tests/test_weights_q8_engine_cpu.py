"""Weights in 8 bits around the kernels, on the CPU: plain statements stand in the kernels' places.  What is compared is the same model whose matrices were rounded
to codes beforehand, run the ordinary way on activations that are rounded to codes in front of every product."""
import json
import os

import pytest
import torch

import q8_linear_refs as refs
from arle_b200 import ops
from arle_b200.cli import build_parser
from arle_b200.engine import ModelRunner, StepEntry
from arle_b200.engine.engine import Engine, EngineOptions
from arle_b200.engine.loading import load_model, random_model
from arle_b200.sampling import SamplingParams
from arle_b200.weights import WeightError, load_weights, write_safetensors
from arle_b200.weights.q8 import StoredQ8, as_q8_weight

E4M3, E8M0 = refs.E4M3, refs.E8M0
CONFIG = {"architectures": ["Qwen3ForCausalLM"], "hidden_size": 160, "intermediate_size": 200, "num_hidden_layers": 2, "num_attention_heads": 4,
          "num_key_value_heads": 2, "head_dim": 32, "vocab_size": 96, "rms_norm_eps": 1e-6, "rope_theta": 1e6, "max_position_embeddings": 256,
          "tie_word_embeddings": True, "bos_token_id": 1, "eos_token_id": 95}


def _put(codes, scales, y):
    c, s = refs.quantize(y)
    codes.copy_(c.to(E4M3)), scales.copy_(s.to(torch.float32).to(E8M0))


def _quantize(x, codes, scales):
    _put(codes, scales, x.double())


def _weight(w, codes, scales):
    c, s = refs.quantize_weight(w.double())
    codes.copy_(c.to(E4M3)), scales.copy_(s)
    return ops.Q8Weight(codes, scales)


def _norm(resid, delta, weight, eps, codes, scales, sum_out=None, delta_scale=1.0):
    x = resid if delta is None else resid + delta_scale * delta.float()
    if sum_out is not None:
        sum_out.copy_(x)
    y = x.double()
    _put(codes, scales, y / (y.square().mean(dim=1, keepdim=True) + eps).sqrt() * weight.double())


def _gemm(codes, scales, w, out):
    out.copy_(refs.product(refs.host(codes), refs.host(scales), refs.host(w.codes), refs.host(w.scales))[0])


def _gated(codes, scales, w, gate_up, out_codes, out_scales, activation="silu"):
    sums = refs.product(refs.host(codes), refs.host(scales), refs.host(w.codes), refs.host(w.scales))[0].view(codes.shape[0], -1, 2, 128)
    _put(out_codes, out_scales, (refs.act(sums[:, :, 0], activation) * sums[:, :, 1]).reshape(codes.shape[0], -1))


@pytest.fixture
def q8_kernels(cpu_kernels, monkeypatch):
    for name, f in (("quantize_q8", _quantize), ("quantize_weight_q8", _weight), ("rmsnorm_q8", _norm), ("gemm_q8", _gemm), ("gemm_act_mul_q8", _gated),
                    ("gate_needs_sums_q8", lambda M, w: M < 3)):
        monkeypatch.setattr(ops, name, f)


def _logits(model, cuts=((0, 9), (9, 10), (10, 40))):
    r = ModelRunner(model, 8, 40, 2, 200, "cpu")
    ids = torch.randint(0, 95, (40,), generator=torch.Generator().manual_seed(4)).tolist()
    return torch.cat([r.step([StepEntry("a", ids[a:b], tuple(range(b - a)))]).clone() for a, b in cuts])


def test_logits_are_those_of_rounded_matrices_and_rows(q8_kernels, monkeypatch):
    model = random_model(CONFIG, 3, "float32", "cpu", sigma=0.1, weight_dtype="float8_e4m3")
    assert model.weight_dtype == "float8_e4m3" and isinstance(model.blocks[0].mixer.w_qkv, ops.Q8Weight)
    got = _logits(model)
    assert (_logits(model, ((0, 40),)) - got).abs().max() < 1e-4          # the same however a prompt is cut

    # the ordinary path on the same numbers: matrices rounded beforehand, rows rounded in front of every product of a block
    wide = random_model(CONFIG, 3, "float32", "cpu", sigma=0.1)
    for b in wide.blocks:
        for part, name in ((b.mixer, "w_qkv"), (b.mixer, "w_o"), (b.ffn, "w_down")):
            w = getattr(part, name)
            setattr(part, name, refs.weight_values(*refs.quantize_weight(w.double()))[:, : w.shape[1]].float())
        g = b.ffn.w_gate_up
        for i in (0, 1):
            g[i::2] = refs.weight_values(*refs.quantize_weight(g[i::2].double()))[:, : g.shape[1]].float()
    plain, gate, head = ops.gemm, ops.gemm_act_mul, wide.head

    def rounded(x):
        return refs.values(*refs.quantize(x.double()))[:, : x.shape[1]].float()

    monkeypatch.setattr(ops, "gemm", lambda x, w, out, sink=None: plain(x if w is head else rounded(x), w, out, sink))
    monkeypatch.setattr(ops, "gemm_act_mul", lambda x, w, gu, out, activation="silu": gate(rounded(x), w, gu, out, activation))
    want = _logits(wide)
    # float32 sums on both sides; a number next to a border between two codes may fall on either side of it, which moves a logit by far less than the rounding
    # itself does (2^-4 of every number)
    assert float((got - want).norm() / want.norm()) < 2e-3


def test_generation(q8_kernels):
    model = random_model(CONFIG, 5, "float32", "cpu", sigma=0.2, weight_dtype="float8_e4m3")
    outs = []
    for chunk in (64, 7):
        eng = Engine(model=model, options=EngineOptions(dtype="float32", device="cpu", page_size=8, num_slots=4, num_pages=60, max_seq_len=128, cuda_graph=False,
                                                        chunked_prefill_size=chunk, weight_dtype="float8_e4m3"))
        outs.append([o.token_ids for o in eng.generate([[5, 9, 17, 33, 2], [7] * 30, [11, 12]], SamplingParams(max_new_tokens=8, ignore_eos=True))])
        eng.runner.cache.check()
    assert outs[0] == outs[1]


def test_what_is_refused(q8_kernels):
    with pytest.raises(ValueError, match="weight_dtype"):
        random_model(CONFIG, 3, "float32", "cpu", weight_dtype="int4")
    model = random_model(CONFIG, 3, "float32", "cpu")
    with pytest.raises(ValueError, match="loaded with weights"):
        Engine(model=model, options=EngineOptions(dtype="float32", device="cpu", weight_dtype="float8_e4m3", num_pages=10, cuda_graph=False))
    from tiny_kolodra import CONFIGS

    with pytest.raises(ValueError, match="pre-norm blocks"):
        random_model(CONFIGS["K1"], 3, "float32", "cpu", weight_dtype="float8_e4m3")


def test_command_line():
    assert build_parser().parse_args(["--weight-dtype", "float8_e4m3"]).weight_dtype == "float8_e4m3"


# ------------------------------------------------------------------ stored codes
def _folder(tmp_path, rows=128):
    """A checkpoint whose layers' matrices are stored as codes with scales that are no powers of two."""
    config = dict(CONFIG, hidden_size=256, head_dim=rows, num_hidden_layers=1)
    wide = random_model(config, 7, "bfloat16", "cpu")
    from arle_b200.weights import random_tensors

    tensors, numbers = {}, {}
    for name, t in random_tensors(wide.weight_decls(), 7, dtype=torch.bfloat16).items():
        if "proj" in name:
            c, s = refs.quantize_weight(t.double())
            s = s * (1.0 + torch.rand(s.shape, generator=torch.Generator().manual_seed(len(name)), dtype=torch.float64)).float().double()
            c = refs.round_e4m3(t.double() / s.repeat_interleave(128, dim=0)[: t.shape[0]].repeat_interleave(128, dim=1)[:, : t.shape[1]])
            tensors[name], tensors[name + "_scale_inv"] = c.to(E4M3), s.float()
            numbers[name] = (c, s)
        else:
            tensors[name] = t
    folder = os.path.join(tmp_path, "stored")
    os.makedirs(folder, exist_ok=True)
    with open(os.path.join(folder, "config.json"), "w") as f:
        json.dump(config, f)
    write_safetensors(os.path.join(folder, "model.safetensors"), tensors)
    return folder, wide, tensors, numbers


def test_stored_codes_are_kept_as_they_are(q8_kernels, tmp_path):
    folder, wide, tensors, numbers = _folder(tmp_path)
    model = load_model(folder, "bfloat16", "cpu", weight_dtype="float8_e4m3")
    mixer, ffn = model.blocks[0].mixer, model.blocks[0].ffn
    prefix = "model.layers.0.self_attn."
    at = 0
    for r in ("q", "k", "v"):
        c, s = numbers[prefix + r + "_proj.weight"]
        n = c.shape[0]
        assert torch.equal(refs.host(mixer.w_qkv.codes[at: at + n, : c.shape[1]]), c) and torch.equal(mixer.w_qkv.scales[at // 128: (at + n) // 128].double(), s)
        at += n
    c, s = numbers["model.layers.0.mlp.down_proj.weight"]
    assert torch.equal(refs.host(ffn.w_down.codes[:, : c.shape[1]]), c) and torch.equal(ffn.w_down.scales.double(), s) and (refs.host(ffn.w_down.codes[:, c.shape[1]:]) == 0).all()
    full = refs.weight_values(refs.host(ffn.w_gate_up.codes), refs.host(ffn.w_gate_up.scales)).view(-1, 2, 128, 256)
    for j, name in enumerate(("gate", "up")):
        c, s = numbers[f"model.layers.0.mlp.{name}_proj.weight"]
        assert torch.equal(full[:, j].reshape(-1, 256)[: c.shape[0]], refs.weight_values(c, s))


def test_stored_codes_as_16_bits(tmp_path):
    folder, wide, tensors, numbers = _folder(tmp_path)
    model = load_model(folder, "bfloat16", "cpu")
    c, s = numbers["model.layers.0.self_attn.o_proj.weight"]
    want = refs.weight_values(c, s)[:, : c.shape[1]] if c.shape[1] % 128 == 0 else None
    assert torch.equal(model.blocks[0].mixer.w_o.double(), want.float().to(torch.bfloat16).double())


def test_stored_matrices_that_end_inside_a_block():
    g = torch.Generator().manual_seed(0)
    parts = [StoredQ8(torch.randn(n, 100, generator=g).to(E4M3), torch.rand(-(-n // 128), 1, generator=g) + 0.5) for n in (128, 130, 5)]
    assert as_q8_weight(parts, "cpu") is None and as_q8_weight(parts[:2], "cpu").shape == (258, 128) and as_q8_weight([parts[0], torch.zeros(1)], "cpu") is None
    want = parts[1].codes.float() * parts[1].scales.repeat_interleave(128, dim=0)[:130]
    assert torch.equal(parts[1].to(dtype=torch.float32), want) and parts[1].to("cpu").dtype == torch.bfloat16
    with pytest.raises(ValueError):
        StoredQ8(parts[0].codes, torch.ones(2, 1))


def test_scales_that_are_missing_or_do_not_fit(tmp_path):
    folder, wide, tensors, _ = _folder(tmp_path)
    name = "model.layers.0.mlp.up_proj.weight"
    for change in (lambda t: t.pop(name + "_scale_inv"), lambda t: t.update({name + "_scale_inv": torch.ones(1, 1)})):
        t = dict(tensors)
        change(t)
        write_safetensors(os.path.join(folder, "model.safetensors"), t)
        with pytest.raises(WeightError, match="_scale_inv"):
            load_weights(folder, wide.weight_decls())

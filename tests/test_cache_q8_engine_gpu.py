"""The operators of the 8-bit cache together, as the engine runs them: tables made on the device, projections, norm and rotation, store, attention, in
portions and decoded tokens, eager and in captured graphs."""
import pytest
import torch

import q8_refs as refs
from arle_b200 import ops
from arle_b200.cache import CacheManager
from arle_b200.engine import ModelRunner, StepEntry
from arle_b200.engine.batch import StepContext, Workspace
from arle_b200.engine.engine import Engine, EngineOptions
from arle_b200.engine.loading import random_model
from arle_b200.parts import build_part
from arle_b200.parts.attention import AttentionSpec
from arle_b200.parts.rotary import RotarySpec
from arle_b200.sampling import SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
F64 = torch.float64
CONFIG = {"architectures": ["Qwen3ForCausalLM"], "hidden_size": 512, "intermediate_size": 1024, "num_hidden_layers": 3, "num_attention_heads": 8,
          "num_key_value_heads": 2, "head_dim": 128, "vocab_size": 1000, "rms_norm_eps": 1e-6, "rope_theta": 1e6, "max_position_embeddings": 4096,
          "tie_word_embeddings": True, "bos_token_id": 1, "eos_token_id": 999}


@pytest.fixture(scope="module")
def model():
    return random_model(CONFIG, 5, "bfloat16", "cuda:0", sigma=0.05)


def _generate(model, dtype="bfloat16", **kw):
    o = dict(dtype=dtype, page_size=16, num_slots=8, num_pages=700, max_seq_len=2048)
    eng = Engine(model=model, options=EngineOptions(**{**o, **kw}))
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 999, (n,), generator=g).tolist() for n in (5, 300, 17, 1000, 64)]
    out = [x.token_ids for x in eng.generate(prompts, SamplingParams(max_new_tokens=40, ignore_eos=True))]
    eng.runner.cache.check()
    return out, eng


def test_tables_on_the_device_change_no_token(model):
    for kw in ({}, {"cache_dtype": "float8_e4m3"}):
        want, host = _generate(model, chunked_prefill_size=256, **kw)
        got, dev = _generate(model, chunked_prefill_size=256, device_tables=True, **kw)
        assert got == want and dev.runner.graph_steps == host.runner.graph_steps > 0
        for g in dev.runner.cache.groups:
            assert (g.device_table.cpu().numpy() < 700).all()


def test_captured_decode_steps_are_the_eager_ones(model):
    want, eager = _generate(model, cache_dtype="float8_e4m3", cuda_graph=False, device_tables=True)
    got, graphs = _generate(model, cache_dtype="float8_e4m3", device_tables=True)
    assert got == want and graphs.runner.graph_steps > 0 == eager.runner.graph_steps


def test_half_the_bytes_of_a_token(model):
    _, eng = _generate(model, cache_dtype="float8_e4m3")
    _, wide = _generate(model)
    assert eng.runner.cache.bytes_per_token() * 2 == wide.runner.cache.bytes_per_token() + 2 * 3 * 2 * 2 * 4 // 16
    auto = Engine(model=model, options=EngineOptions(cache_dtype="float8_e4m3", num_slots=4, max_seq_len=512, mem_fraction_static=0.5))      # pages from free memory
    assert auto.runner.cache.total_pages() == [4 * 512 // 16]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_of_the_kernel_sets_and_of_a_wide_cache(dtype):
    """e4m3 against the wide cache: a key or value is off by at most 2^-4 of itself, so the logits stay within a tenth of their norm (they would not, were a
    page, a scale or a place wrong).  Between the kernel sets a float32 projection differs in its last bits (2^-22 of it, say), which moves one number in
    2^22 / 2^4 or so, of the 700 * 512 * 3 stored here a few, across a border between two codes, by a step of 2^-3 at most: the sets are off
    each other by less than the rounding to codes, which moves every number by up to 2^-4, is off the wide cache."""
    model = random_model(CONFIG, 6, dtype, "cuda:0", sigma=0.05)
    ids = torch.randint(0, 999, (700,), generator=torch.Generator().manual_seed(2)).tolist()

    def run(**kw):
        r = ModelRunner(model, 16, 60, 2, 800, "cuda:0", **kw)
        out = [r.step([StepEntry("a", ids[a:b], tuple(range(b - a)))]).clone() for a, b in ((0, 333), (333, 334), (334, 336), (336, 700))]
        ops.check_errors(DEV)
        return torch.cat(out)

    wide, q8, plain = run(), run(cache_dtype=E4M3), run(cache_dtype=E4M3, kernel_set="plain")
    assert (q8 - wide).norm() <= 0.1 * wide.norm()
    assert (q8 - plain).norm() <= (0.03 * plain.norm() if dtype == torch.bfloat16 else 0.1 * (q8 - wide).norm())


@pytest.mark.parametrize("window", [None, 48])
def test_an_attention_layer_step_by_step(window):
    """A layer over three requests, cut at odd places, 60 decode steps: every step's output against 64 bits from the layer's own projections, the cache
    against the store's definition."""
    nq, nkv, hd, H, ps = 8, 2, 128, 256, 16
    part = build_part(AttentionSpec("", H, nq, nkv, hd, hd ** -0.5, 1e-6, RotarySpec(hd, 1e4), window=window))
    g = torch.Generator().manual_seed(3)
    part.load({d.name: torch.randn(d.shape, generator=g) * (0.1 if len(d.shape) == 2 else 0.0) + (len(d.shape) == 1) for d in part.weight_decls()}, torch.bfloat16, DEV)
    cm = CacheManager([part.cache_need()], [], ps, 60, 4, 400, torch.bfloat16, DEV, cache_dtype=E4M3, device_tables=window is None)
    ctx = StepContext(cm, Workspace(DEV))
    for rid in "abc":
        cm.add_request(rid)
    plan = [[("a", 37)], [("b", 100), ("a", 1)], [("c", 5), ("a", 20), ("b", 1)]] + [[("a", 1), ("b", 1), ("c", 1)]] * 60
    codes, scales = [torch.zeros_like(x[0], dtype=F64, device="cpu") for x in cm.groups[0].arrays], [torch.zeros_like(x[0], dtype=F64, device="cpu") for x in cm.groups[0].scales]
    for step, items in enumerate(plan):
        starts = [cm.num_tokens(r) for r, _ in items]
        cm.append(items)
        ctx.build([StepEntry(r, [0] * n) for r, n in items], starts)
        view, T = ctx.cache_view(0), ctx.num_tokens
        x = torch.randn(T, H, generator=g).bfloat16().to(DEV)
        out = part.forward(x, ctx, view, None).clone()
        proj = ctx.ws.get("qkv", (T, (nq + 2 * nkv) * hd), torch.bfloat16)          # normed and turned in place
        slots = view.slot_mapping.tolist()
        for i, at in ((0, nq), (1, nq + nkv)):
            refs.store(proj[:, at * hd: (at + nkv) * hd].double().cpu().view(T, nkv, hd), slots, codes[i], scales[i])
            assert torch.equal(view.scales[i].double().cpu(), scales[i])
            assert torch.equal(view.streams[i].float().double().cpu(), codes[i])
        want, size, big = refs.attention(proj[:, : nq * hd], view.k.float(), view.v.float(), *view.scales, ctx.q_indptr.tolist(), ctx.kv_lens.tolist(), view.block_table,
                                         nq, nkv, hd ** -0.5, window, None)
        attn = ctx.ws.get("attn_out", (T, nq * hd), torch.bfloat16)
        # weights rounded to bfloat16 at the coarsest, scores off by 2^-13 at most (see test_attention_q8_gpu.py), the result's rounding
        assert ((attn.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + size * (2.0 ** -8 + 2.0 ** -12 * (1 + big))).all()
        ref = attn.double() @ part.w_o.double().T
        assert (out.double() - ref).norm() <= 2.0 ** -7 * ref.norm()
        for r, _ in items:
            cm.release_passed(r)
    ops.check_errors(DEV)

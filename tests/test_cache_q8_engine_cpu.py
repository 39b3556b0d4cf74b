"""The 8-bit cache and tables made on the device around the kernels, on the CPU: plain statements (tests/q8_refs.py) stand in the kernels' places."""
import numpy as np
import pytest
import torch

import q8_refs as refs
from arle_b200 import ops
from arle_b200.cache import CacheManager
from arle_b200.engine import ModelRunner, StepEntry
from arle_b200.engine.engine import Engine, EngineOptions
from arle_b200.engine.batch import StepContext, Workspace
from arle_b200.engine.loading import random_model
from arle_b200.parts.base import CacheNeed
from arle_b200.sampling import SamplingParams

E4M3 = torch.float8_e4m3fn
CONFIG = {"architectures": ["Qwen3ForCausalLM"], "hidden_size": 32, "intermediate_size": 48, "num_hidden_layers": 2, "num_attention_heads": 4,
          "num_key_value_heads": 2, "head_dim": 16, "vocab_size": 96, "rms_norm_eps": 1e-6, "rope_theta": 1e6, "max_position_embeddings": 256,
          "tie_word_embeddings": True, "bos_token_id": 1, "eos_token_id": 95}


def _store(k, v, slot_mapping, k_cache, v_cache, k_scale, v_scale, nkv, hd, page_size, vd=None):
    for x, c, s in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        c64, s64 = c.float().double(), s.double()
        refs.store(x.double().reshape(x.shape[0], nkv, -1), slot_mapping.tolist(), c64, s64)
        c.copy_(c64.float())
        s.copy_(s64)


def _attend(q, out, k_cache, v_cache, k_scale, v_scale, positions, row_of_token, block_table, nq, nkv, hd, page_size, scale, window, batch=None, vd=None, sink=None):
    o, _, _ = refs.attention(q, k_cache.float(), v_cache.float(), k_scale, v_scale, batch.q_indptr.tolist(), batch.kv_lens.tolist(), block_table, nq, nkv, scale, window,
                             sink)
    out.copy_(o)


def _tables(slots, starts, q_lens, new_pages, page_table, num_pages, page_size, q_indptr, kv_lens, positions, row_of_token, slot_of_token, slot_mapping, block_table, status):
    table = page_table.tolist()
    got = refs.tables(slots.tolist(), starts.tolist(), q_lens.tolist(), new_pages.tolist(), table, page_size, block_table.shape[1])
    for t, x in zip((q_indptr, kv_lens, positions, row_of_token, slot_of_token, slot_mapping, block_table, page_table), got + (table,)):
        t.copy_(torch.tensor(x, dtype=torch.int32))
    status.zero_()


@pytest.fixture
def q8_kernels(cpu_kernels, monkeypatch):
    for name, f in (("store_q8", _store), ("paged_attention_q8", _attend), ("step_tables", _tables)):
        monkeypatch.setattr(ops, name, f)


@pytest.fixture(scope="module")
def model():
    return random_model(CONFIG, 3, "float32", "cpu", sigma=0.2)


def _generate(model, **kw):
    eng = Engine(model=model, options=EngineOptions(dtype="float32", device="cpu", page_size=8, num_slots=4, num_pages=60, max_seq_len=128, cuda_graph=False, **kw))
    prompts = [[5, 9, 17, 33, 2], [7] * 30, [11, 12]]
    out = [o.token_ids for o in eng.generate(prompts, SamplingParams(max_new_tokens=12, ignore_eos=True))]
    eng.runner.cache.check()
    return out, eng


def test_tables_on_the_device_change_nothing(model, q8_kernels):
    want, host = _generate(model, chunked_prefill_size=7)
    got, eng = _generate(model, chunked_prefill_size=7, device_tables=True)
    assert got == want and eng.runner.ctx.h2d_bytes < host.runner.ctx.h2d_bytes
    with pytest.raises(ValueError, match="wanted place"):
        eng.runner.step([StepEntry("x", [1, 2], (2,))])


def test_generation_on_an_8_bit_cache(model, q8_kernels):
    got, eng = _generate(model, cache_dtype="float8_e4m3")
    assert [len(x) for x in got] == [12, 12, 12]
    g = eng.runner.cache.groups[0]
    assert g.arrays[0].dtype == E4M3 and g.scales[0].shape == (2, 60, 2)
    assert eng.runner.cache.bytes_per_token() == 2 * (2 * 2 * 16 * 8 + 4 * 4) // 8
    both, _ = _generate(model, cache_dtype="float8_e4m3", device_tables=True)
    assert both == got


def test_logits_on_an_8_bit_cache(model, q8_kernels):
    """Against the same model on a float32 cache: e4m3 is off by at most 2^-4 of a number, so keys and values are, and logits stay near."""
    ids = list(np.random.default_rng(0).integers(0, 95, 40))
    logits = []
    for kw in ({}, {"cache_dtype": E4M3}):
        r = ModelRunner(model, 8, 20, 2, 100, "cpu", **kw)
        logits.append(torch.cat([r.step([StepEntry("a", ids[a:b], tuple(range(b - a)))]).clone() for a, b in ((0, 13), (13, 14), (14, 40))]))
    off = (logits[1] - logits[0]).norm() / logits[0].norm()
    assert 0 < off < 0.1


def test_what_is_refused(model):
    with pytest.raises(ValueError, match="cache_dtype"):
        Engine(model=model, options=EngineOptions(dtype="float32", device="cpu", cache_dtype="int8", cuda_graph=False, num_pages=4))
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        CacheManager([CacheNeed(1, 8)], [], 8, 4, 2, 32, torch.float32, "cpu", cache_dtype=torch.bfloat16)
    for need in (CacheNeed(1, 8, window=16), CacheNeed(1, 8, chunk=16)):
        with pytest.raises(ValueError, match="window"):
            CacheManager([need], [], 8, 4, 2, 32, torch.float32, "cpu", device_tables=True)
    with pytest.raises(ValueError, match="4,096"):
        CacheManager([CacheNeed(1, 8)], [], 8, 4, 5000, 32, torch.float32, "cpu", device_tables=True)

    class Other:
        def cache_need(self):
            return CacheNeed(1, 8)

        def takes_q8_cache(self):
            return False

    class Blocks:
        blocks = [type("B", (), {"mixer": Other()})()]

    with pytest.raises(ValueError, match="Other"):
        ModelRunner(Blocks(), 8, 4, 2, 32, "cpu", cache_dtype=E4M3)


def test_a_step_that_fails_is_forgotten_on_the_device_too(q8_kernels):
    cm = CacheManager([CacheNeed(1, 8), CacheNeed(2, 8)], [], 4, 9, 3, 24, torch.float32, "cpu", device_tables=True)
    ctx = StepContext(cm, Workspace("cpu"))
    for rid in "ab":
        cm.add_request(rid)

    def step(items):
        starts = [cm.num_tokens(r) for r, _ in items]
        cm.append(items)
        ctx.build([StepEntry(r, [0] * n) for r, n in items], starts)

    step([("a", 6), ("b", 3)])
    cm.append([("a", 9)])
    cm.truncate("a", 6)                    # pages of a step that failed go back, and another request gets them
    step([("b", 8)])
    step([("a", 7), ("b", 1)])
    for gi, g in enumerate(cm.groups):
        for rid in "ab":
            n = -(-cm.num_tokens(rid) // 4)
            assert g.device_table[cm.slot(rid), :n].tolist() == g.table[cm.slot(rid), :n].tolist()
        assert ctx.groups[gi].slot_mapping.tolist() == cm.slot_mapping(gi, "a", 6, 7).tolist() + cm.slot_mapping(gi, "b", 11, 1).tolist()
        assert ctx.groups[gi].block_table.tolist() == cm.block_rows(gi, ["a", "b"]).tolist()

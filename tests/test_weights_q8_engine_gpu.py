"""Weights in 8 bits in the engine: norm, products, gate and codes together, in portions and decoded tokens, eager and in captured graphs."""
import pytest
import torch

from arle_b200 import ops
from arle_b200.engine import ModelRunner, StepEntry
from arle_b200.engine.engine import Engine, EngineOptions
from arle_b200.engine.loading import random_model
from arle_b200.sampling import SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CONFIG = {"architectures": ["Qwen3ForCausalLM"], "hidden_size": 512, "intermediate_size": 1100, "num_hidden_layers": 3, "num_attention_heads": 8,
          "num_key_value_heads": 2, "head_dim": 128, "vocab_size": 1000, "rms_norm_eps": 1e-6, "rope_theta": 1e6, "max_position_embeddings": 4096,
          "tie_word_embeddings": True, "bos_token_id": 1, "eos_token_id": 999}


@pytest.fixture(scope="module")
def model():
    return random_model(CONFIG, 5, "bfloat16", DEV, sigma=0.05, weight_dtype="float8_e4m3")


def _generate(model, **kw):
    o = dict(page_size=16, num_slots=8, num_pages=700, max_seq_len=2048, weight_dtype="float8_e4m3")
    eng = Engine(model=model, options=EngineOptions(**{**o, **kw}))
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 999, (n,), generator=g).tolist() for n in (5, 300, 17, 1000, 64)]
    out = [x.token_ids for x in eng.generate(prompts, SamplingParams(max_new_tokens=40, ignore_eos=True))]
    eng.runner.cache.check()
    return out, eng


@pytest.mark.parametrize("kw", [{}, {"cache_dtype": "float8_e4m3"}])
def test_captured_decode_steps_are_the_eager_ones(model, kw):
    want, eager = _generate(model, cuda_graph=False, **kw)
    got, graphs = _generate(model, **kw)
    assert got == want and graphs.runner.graph_steps > 0 == eager.runner.graph_steps


def test_two_engines_with_captured_steps_side_by_side(model):
    """Two engines on the same weights, their captured steps in turn: neither finds the other's numbers in its buffers."""
    want, _ = _generate(model)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 999, (n,), generator=g).tolist() for n in (5, 300, 17, 1000, 64)]
    engines = [Engine(model=model, options=EngineOptions(page_size=16, num_slots=8, num_pages=700, max_seq_len=2048)) for _ in range(2)]
    sp = SamplingParams(max_new_tokens=40, ignore_eos=True)
    reqs = [[e.add_request(p, sp) for p in (prompts if i == 0 else prompts[::-1])] for i, e in enumerate(engines)]
    while any(r.finish_reason is None for rs in reqs for r in rs):
        for e in engines:
            e.step() if e.scheduler.has_work() else e._drain()
    assert [r.output for r in reqs[0]] == want
    assert [len(r.output) for r in reqs[1]] == [40] * 5


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_logits(dtype):
    """A layer's matrices and the rows in front of them are rounded to four bits (2^-4 of a number at most, half of that on average), so logits stay within a
    fifth of those of the wide model; the kernel sets differ by the last bits of float32 sums, which move a few numbers across a border between two codes."""
    wide, q8 = (random_model(CONFIG, 6, dtype, DEV, sigma=0.05, weight_dtype=w) for w in ("auto", "float8_e4m3"))
    ids = torch.randint(0, 999, (700,), generator=torch.Generator().manual_seed(2)).tolist()

    def run(model, **kw):
        r = ModelRunner(model, 16, 60, 2, 800, DEV, **kw)
        out = [r.step([StepEntry("a", ids[a:b], tuple(range(b - a)))]).clone() for a, b in ((0, 333), (333, 334), (334, 360), (360, 420), (420, 700))]
        ops.check_errors(DEV)
        return torch.cat(out)

    a, b, c = run(wide), run(q8), run(q8, kernel_set="plain")
    off = float((b - a).norm() / a.norm())
    assert 1e-3 < off < 0.2, off
    assert float((b - c).norm() / c.norm()) < off / 2


def test_bytes(model):
    """Half of the layers' matrices, and their scales."""
    wide = random_model(CONFIG, 5, "bfloat16", DEV, sigma=0.05)
    head = wide.head.numel() * 2
    assert model.weight_bytes_per_step() - head < 0.56 * (wide.weight_bytes_per_step() - head)          # 1,100 rows are filled up to 1,152

"""A step whose tables the device found out of order: the engine raises before it books the step's tokens.  On the CPU, with a plain statement in the
kernel's place."""
import pytest
import torch

import test_cache_q8_engine_cpu as plain
from arle_b200 import ops
from arle_b200.cache import CacheManager
from arle_b200.engine import StepEntry
from arle_b200.engine.batch import StepContext, Workspace
from arle_b200.engine.engine import Engine, EngineOptions
from arle_b200.parts.base import CacheNeed
from arle_b200.sampling import SamplingParams

model = plain.model


@pytest.fixture
def fail_at(cpu_kernels, monkeypatch):
    """Calls of ``step_tables`` (counted from 0) that say of themselves that a step is not in order."""
    calls, bad = [0], {}

    def tables(*args):
        plain._tables(*args)
        args[-1].fill_(bad.get(calls[0], 0))
        calls[0] += 1

    monkeypatch.setattr(ops, "step_tables", tables)
    return bad


@pytest.mark.parametrize("at", [0, 1, 5, 12])
def test_the_engine_raises_before_it_books_the_tokens(model, fail_at, at):
    """The first step, one in the middle, and the last (a prompt and 12 tokens, none after the 13th call)."""
    fail_at[at] = 8
    eng = Engine(model=model, options=EngineOptions(dtype="float32", device="cpu", page_size=8, num_slots=4, num_pages=60, max_seq_len=128, cuda_graph=False,
                                                    device_tables=True))
    seen = []
    with pytest.raises(RuntimeError, match="status 8"):
        eng.generate([[5, 9, 17]], SamplingParams(max_new_tokens=13, ignore_eos=True), on_token=lambda rid, t: seen.append(t))
    assert len(seen) == at


def test_every_group_has_a_word_of_its_own(fail_at):
    """Two cache groups: the first one's failure is not lost to the second one's success, and the step after it does not run."""
    fail_at[2] = 4
    cm = CacheManager([CacheNeed(1, 8), CacheNeed(2, 8)], [], 4, 9, 3, 24, torch.float32, "cpu", device_tables=True)
    ctx = StepContext(cm, Workspace("cpu"))
    cm.add_request("a")

    def step(n):
        start = cm.num_tokens("a")
        cm.append([("a", n)])
        ctx.build([StepEntry("a", [0] * n)], [start])

    step(3)
    ctx.tables_status.check()
    step(2)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="group 0.*status 4"):
            ctx.tables_status.check()
    with pytest.raises(RuntimeError, match="group 0"):
        step(1)


def test_a_step_of_the_hosts_tables_has_no_status(cpu_kernels):
    cm = CacheManager([CacheNeed(1, 8)], [], 4, 9, 3, 24, torch.float32, "cpu")
    ctx = StepContext(cm, Workspace("cpu"))
    cm.add_request("a")
    cm.append([("a", 3)])
    ctx.build([StepEntry("a", [0] * 3)], [0])
    assert ctx.tables_status is None

"""Tables made on the device for requests whose room was made without a step.  On the CPU, with a plain statement in the kernel's place."""
import numpy as np
import pytest
import torch

import test_cache_q8_engine_cpu as plain
from arle_b200 import ops
from arle_b200.cache import CacheManager
from arle_b200.engine import StepEntry
from arle_b200.engine.batch import StepContext, Workspace
from arle_b200.parts.base import CacheNeed


@pytest.fixture
def made(cpu_kernels, monkeypatch):
    monkeypatch.setattr(ops, "step_tables", plain._tables)
    cm = CacheManager([CacheNeed(1, 8), CacheNeed(2, 8)], [], 4, 30, 3, 40, torch.float32, "cpu", device_tables=True)
    ctx = StepContext(cm, Workspace("cpu"))

    def step(items):
        starts = [cm.num_tokens(r) for r, _ in items]
        cm.append(items)
        ctx.build([StepEntry(r, [0] * n) for r, n in items], starts)
        for gi, g in enumerate(cm.groups):
            for row, (rid, n) in enumerate(items):
                pages = -(-cm.num_tokens(rid) // 4)
                host = g.table[cm.slot(rid), :pages].tolist()
                assert ctx.groups[gi].block_table[row, :pages].tolist() == host and g.device_table[cm.slot(rid), :pages].tolist() == host
            want = np.concatenate([cm.slot_mapping(gi, rid, s, n) for (rid, n), s in zip(items, starts)])
            assert ctx.groups[gi].slot_mapping.tolist() == want.tolist()

    return cm, step


def test_room_in_front_of_the_first_step(made):
    cm, step = made
    cm.add_request("a"), cm.add_request("b")
    cm.append([("a", 11)])
    step([("a", 1), ("b", 5)])
    step([("a", 1), ("b", 1)])


def test_room_between_steps(made):
    cm, step = made
    cm.add_request("a")
    step([("a", 6)])
    cm.append([("a", 9)])
    step([("a", 2)])


def test_room_that_was_given_back_and_taken_again(made):
    """A request is cut back to a page's end and grows without a step; another one has its old pages by then."""
    cm, step = made
    cm.add_request("a"), cm.add_request("b")
    step([("a", 16), ("b", 1)])
    cm.truncate("a", 8)
    step([("b", 12)])
    cm.append([("a", 9)])
    step([("a", 3), ("b", 1)])


def test_a_slot_that_another_request_had(made):
    cm, step = made
    cm.add_request("a")
    step([("a", 16)])
    cm.free_request("a")
    cm.add_request("b")
    cm.append([("b", 14)])
    step([("b", 1)])

"""A step's tables made on the GPU, whole numbers against the definition."""
import math

import pytest
import torch

import q8_refs as refs
from arle_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _outs(R, T, width):
    o = {n: torch.full((k,), -7, dtype=torch.int32, device=DEV)
         for n, k in (("q_indptr", R + 1), ("kv_lens", R), ("positions", T), ("row_of_token", T), ("slot_of_token", T), ("slot_mapping", T))}
    o["block_table"] = torch.full((R, width), -7, dtype=torch.int32, device=DEV)
    o["status"] = torch.full((1,), -7, dtype=torch.int32, device=DEV)
    return o


def _call(slots, starts, lens, new, table, num_pages, ps, o):
    ops.step_tables(_i32(slots), _i32(starts), _i32(lens), _i32(new), table, num_pages, ps, o["q_indptr"], o["kv_lens"], o["positions"], o["row_of_token"],
                    o["slot_of_token"], o["slot_mapping"], o["block_table"], o["status"])


def _make(rows, ps, slots, most, news, seed):
    g = torch.Generator().manual_seed(seed)
    draw = lambda hi: int(torch.randint(0, hi + 1, (1,), generator=g))      # noqa: E731
    starts, lens = [draw(most) for _ in range(rows)], [draw(news) if news > 1 else 1 for _ in range(rows)]
    ids = torch.randperm(slots, generator=g).tolist()[:rows]
    held = [math.ceil(s / ps) for s in starts]
    need = [math.ceil((s + n) / ps) for s, n in zip(starts, lens)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).tolist()
    width = max(need + [1])
    table, at = [[-1] * (width + 2) for _ in range(slots)], 0
    for i, h in zip(ids, held):
        table[i][:h] = order[at: at + h]
        at += h
    return ids, starts, lens, order[at: sum(need)], table, pages, width


@pytest.mark.parametrize("rows,ps,slots,most,news", [(1, 16, 1, 0, 1), (1, 16, 3, 40, 1), (8, 16, 64, 2000, 1), (5, 1, 9, 30, 7), (33, 7, 40, 300, 60), (600, 16, 700, 500, 1),
                                                     (513, 64, 513, 900, 40), (3, 16, 4, 20000, 9000), (4096, 16, 65536, 40, 3)])
def test_tables(rows, ps, slots, most, news):
    for seed in range(3):
        ids, starts, lens, new, table, pages, width = _make(rows, ps, slots, most, news, seed)
        T = sum(lens)
        o = _outs(rows, T + 5, width + 1)                       # five tokens more than the step has
        dev = _i32(table)
        _call(ids, starts, lens, new, dev, pages, ps, o)
        indptr, kv, pos, row, sl, place, blocks = refs.tables(ids, starts, lens, new, table, ps, width + 1)
        assert int(o["status"]) == 0
        assert o["q_indptr"].tolist() == indptr and o["kv_lens"].tolist() == kv
        for name, want in (("positions", pos), ("row_of_token", row), ("slot_of_token", sl), ("slot_mapping", place)):
            assert o[name].tolist() == want + [-7] * 5, name
        assert o["block_table"].tolist() == blocks and dev.tolist() == table
        _call(ids, starts, lens, new, dev, pages, ps, o)        # the same step again: the same tables
        assert o["block_table"].tolist() == blocks and dev.tolist() == table


@pytest.mark.parametrize("what,bit", [("tokens", 1), ("twice", 2), ("slot", 2), ("low slot", 2), ("long", 4), ("few", 8), ("negative", 16), ("start", 16), ("foreign", 32),
                                      ("low page", 32)])
def test_a_step_that_is_not_in_order_is_left_out(what, bit):
    ids, starts, lens, ps = [2, 0, 5], [10, 0, 33], [3, 40, 1], 16
    new = [7, 8, 9]
    table = [[-1] * 4 for _ in range(6)]
    table[2][0], table[5][:3] = 1, [2, 3, 4]
    T = 44
    if what == "tokens":
        T = 43
    elif what == "twice":
        ids[1] = 2
    elif what == "slot":
        ids[0] = 6
    elif what == "low slot":
        ids[2] = -1
    elif what == "long":
        lens[0], T = 80, 200
    elif what == "few":
        new = new[:2]
    elif what == "negative":
        lens[2] = -1
    elif what == "start":
        starts[2] = -5
    elif what == "foreign":
        new[1] = 11
    elif what == "low page":
        new[0] = -1
    o = _outs(3, T, 4)
    dev = _i32(table)
    _call(ids, starts, lens, new, dev, 11, ps, o)
    assert int(o["status"]) & bit and dev.tolist() == table
    assert not o["q_indptr"].any() and not o["kv_lens"].any()
    assert (o["slot_mapping"] == -1).all() and (o["block_table"] == -1).all()
    assert not o["positions"].any() and not o["row_of_token"].any() and not o["slot_of_token"].any()


def test_lengths_near_the_end_of_32_bits():
    o = _outs(2, 10, 4)
    dev = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    for starts, lens in (([2 ** 31 - 1, 0], [2 ** 31 - 1, 1]), ([0, 0], [2 ** 31 - 1, 2 ** 31 - 1])):
        _call([0, 1], starts, lens, [0, 1], dev, 4, 16, o)
        assert int(o["status"]) & 4 and not o["kv_lens"].any() and (dev == -1).all()

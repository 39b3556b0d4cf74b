"""Pages that a request is said to hold and that the cache does not have."""
import pytest
import torch

import test_step_tables_gpu as plain

pytestmark = pytest.mark.gpu


def test_held_pages_outside_the_cache_are_no_pages():
    """Row 0's table names pages behind and in front of the cache; row 1 is as it should be."""
    ps, pages = 4, 9
    table = plain._i32([[2, 9, 2 ** 30, -7, 5, -1], [3, 1, -1, -1, -1, -1]])
    o = plain._outs(2, 5, 6)
    plain._call([0, 1], [20, 7], [2, 3], [6, 8], table, pages, ps, o)
    assert o["status"].item() == 0
    assert o["block_table"].tolist() == [[2, -1, -1, -1, 5, 6], [3, 1, 8, -1, -1, -1]]
    assert o["slot_mapping"].tolist() == [24, 25, 7, 32, 33]
    plain._call([0, 1], [15, 7], [1, 1], [], table, pages, ps, o)      # the next token would go to a page that is not there
    assert o["slot_mapping"].tolist()[:2] == [-1, 7]

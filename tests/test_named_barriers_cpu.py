"""Kernels whose bounded waits may run out: a named barrier (bar.sync of some warps) has no limit of its own, so a warp that gives up still comes to every such barrier
that the warps beside it may go to.  It is one warp that gives up: another's poll of the same mbarrier may succeed a moment later."""
import os
import re

import pytest

from arle_b200.ops import build


def _text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(build.CSRC, name)).read())


def _branch(text, at):
    """The braces' content that starts behind ``at``."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start + 1: i]
    raise AssertionError("braces do not close")


def test_few_rows_a_warp_that_gives_up_comes_to_the_others_barriers():
    text = _text("gemm_q8_few.cu")
    wait = text.index("mbar_wait_bounded(acc_full0")          # the adding warps' wait; their barrier is the one of bar_adders
    given_up = _branch(text, text.index(")", text.index("aborted", wait)))
    assert "bar_adders();" in given_up and given_up.rstrip().endswith("break;")


def test_gates_a_warp_that_gives_up_comes_to_its_partners_barriers():
    text = _text("gemm_q8_tc.cu")
    given_up = _branch(text, text.index("if (lost) {"))
    assert given_up.count("bar_pair(") == 2 and "GATED" in given_up and given_up.rstrip().endswith("break;")


# ------------------------------------------------------------------ the loops as a model: every warp comes to a barrier the same number of times, wherever it gives up
def _adder(blocks, scaled, gives_up_at):
    """Barriers an adding warp of the kernel for few rows comes to; it gives up at the given block (None: never)."""
    count = 0
    for done in range(blocks):
        if done % scaled == 0:
            count += 1
        if done == gives_up_at:
            count += sum(later % scaled == 0 for later in range(done + 1, blocks))
            break
    return count


def _gate(tiles, gives_up_in):
    """The same of an epilogue warp of the gated kernel, two barriers a tile; it gives up in a tile's sums."""
    count = 0
    for t in range(tiles):
        if t == gives_up_in:
            count += sum(2 for _ in range(t, tiles))
            break
        count += 2
    return count


@pytest.mark.parametrize("scaled", [4, 8, 16])
@pytest.mark.parametrize("blocks", [1, 3, 4, 5, 16, 17, 131])
def test_adders_meet(blocks, scaled):
    assert {_adder(blocks, scaled, at) for at in [None, *range(blocks)]} == {-(-blocks // scaled)}


@pytest.mark.parametrize("tiles", [1, 2, 7])
def test_partners_meet(tiles):
    assert {_gate(tiles, at) for at in [None, *range(tiles)]} == {2 * tiles}

"""Kernels that store into the shared memory of other blocks of their cluster: such a store stands behind a wait for the word of every block that it has started.  (Blocks
of a cluster run at the same time; that does not say that each has begun when another stores, and a store before that has no defined effect.)"""
import os
import re

import pytest

from arle_b200.ops import build


def _kernels(name):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(build.CSRC, name)).read())
    starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
    for a, b in zip(starts, starts[1:]):
        yield text[a:b]


def _paths(body):
    """The kernel's text for one and for two blocks of columns, where it has both (the other side of each such condition taken out)."""
    if "NB" not in body:
        return [body]
    one = re.sub(r"if \(NB == 2\) cluster_sync_all\(\);", "", body)
    two = re.sub(r"(?:else|if \(NB == 1[^)]*\)) cluster_(?:all_)?started\(\);", "", body)
    return [one, two]


FILES = [f for f in build.sources() if "st.shared::cluster" in open(os.path.join(build.CSRC, f)).read()]


@pytest.mark.parametrize("name", FILES)
def test_stores_to_other_blocks_wait_for_their_start(name):
    seen = 0
    for kernel in _kernels(name):
        if "store_cluster(" not in kernel:
            continue
        for body in _paths(kernel):
            ahead, behind = body.split("store_cluster(", 1)
            word, wait = ahead.find("cluster_started();"), ahead.find("cluster_all_started();")
            both = ahead.find("cluster_sync_all();")
            assert both >= 0 or 0 <= word < wait, f"{name}: a store to another block without a wait for its start"
            # the word is given before the sums, so that the wait behind them is short, and the wait's own pair is whole: no other barrier of the cluster between
            assert both >= 0 or (word < ahead.find("pdl_wait();") and "cluster_sync_all();" not in ahead[word:wait])
            assert "cluster_sync_all();" in behind, f"{name}: nothing says when the sums are there"
            seen += 1
    assert seen > 0


def test_there_are_such_kernels():
    assert set(FILES) >= {"gemm_q8_few.cu", "gemm_q8_split.cu"}

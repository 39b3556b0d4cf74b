"""Products of 8-bit codes that start beside the kernel in front of them: what that kernel may be writing, the weight's codes among it, is read behind the wait for it.
(Bringing lines to L2 is no reading: it is where memory is the same for all.)"""
import os
import re

import pytest

from arle_b200.ops import build

FILES = [f for f in build.sources() if f.startswith("gemm_q8")]


def _ahead(name):
    """What every kernel of a file does in front of its wait, without comments and without the bodies of functions that are only defined there."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(build.CSRC, name)).read())
    for m in re.finditer(r"__global__.*?pdl_wait\(\);", text, flags=re.S):
        yield re.sub(r"auto \w+ = \[&\]\([^)]*\) \{.*?\n  \};", "", m.group(0), flags=re.S)


@pytest.mark.parametrize("name", FILES)
def test_nothing_is_loaded_in_front_of_the_wait(name):
    seen = list(_ahead(name))
    assert seen
    for ahead in seen:
        assert not re.search(r"\b(tma_load_\w+|load_once|ask|__ld\w+)\(", ahead), f"{name}: loads in front of pdl_wait"


def test_all_products():
    assert set(FILES) == {"gemm_q8.cu", "gemm_q8_few.cu", "gemm_q8_split.cu", "gemm_q8_tc.cu"}


@pytest.mark.parametrize("name", FILES + ["linear_q8.cu"])
def test_operands_are_read_by_plain_loads(name):
    """A kernel that may live beside the one in front of it (all of these, when programmatic launches are on) reads what that one writes by plain loads: not by the way for
    memory that nobody writes meanwhile, which the compiler takes for pointers that are const and restrict."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(build.CSRC, name)).read())
    assert not re.search(r"const\s+\w+\s*\*\s*__restrict__|__ldg\(|ld\.global\.nc", text)

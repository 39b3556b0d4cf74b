"""Caches of more places than 32 bits number are refused when they are made, not at every step."""
import pytest
import torch

from arle_b200.cache import CacheManager
from arle_b200.parts.base import CacheNeed


@pytest.mark.parametrize("kw", [dict(cache_dtype=torch.float8_e4m3fn), dict(device_tables=True)])
def test_more_places_than_32_bits_number(kw):
    make = lambda pages: CacheManager([CacheNeed(1, 8)], [], 2 ** 20, pages, 2, 32, torch.bfloat16, "meta", **kw)      # noqa: E731
    with pytest.raises(ValueError, match="32 bits"):
        make(2 ** 11)
    assert make(2 ** 11 - 1).total_pages() == [2 ** 11 - 1]

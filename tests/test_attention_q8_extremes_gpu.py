"""Attention over the 8-bit cache at the ends of what a cache may hold, against its definition in 64 bits; tolerances as in test_attention_q8_gpu.py."""
import pytest

from test_attention_q8_gpu import _case, _near, _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [False])
def test_values_near_the_largest_number(batch):
    """Values of up to 448 * 2^119: their mean is a number, so their sum must not be an infinity on the way there."""
    s = _case([(1, 900), (1, 40)], 8, 2, 128, 16, seed=13)
    s.vs.fill_(2.0 ** 119)
    s.ks.fill_(2.0 ** -9)
    _near(_run(s, batch=batch), _want(s), 128, 2.0 ** -11 if batch else 0.0, 900)

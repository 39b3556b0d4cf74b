"""Attention over the 8-bit cache at the ends of what a cache may hold, against its definition in 64 bits; tolerances as in test_attention_q8_gpu.py."""
import pytest
import torch

from test_attention_q8_gpu import DEV, E4M3, _case, _near, _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [False, True])
def test_values_near_the_largest_number(batch):
    """Values of up to 448 * 2^119: their mean is a number, so their sum must not be an infinity on the way there."""
    s = _case([(1, 900), (1, 40)], 8, 2, 128, 16, seed=13)
    s.vs.fill_(2.0 ** 119)
    s.ks.fill_(2.0 ** -9)
    _near(_run(s, batch=batch), _want(s), 128, 2.0 ** -11 if batch else 0.0, 900)


@pytest.mark.parametrize("hd,ps", [(64, 16), (128, 16), (128, 12), (64, 20)])
@pytest.mark.parametrize("big,gap", [(23, 60), (23, 133), (119, 60), (119, 133)])
@pytest.mark.parametrize("sink", [None, 95.0])
def test_a_page_of_zeros_has_the_highest_scores(hd, ps, big, gap, sink):
    """A page of zeros has the scale 2^-100; other pages' values are up to 2^30 or 2^127, their scores some 60 or 133 (in log2) below: their weights are
    2^-133 of the largest and carry the whole result.  In front and behind, for the same warp and for others.  (In the general kernel weights are float32 numbers
    by themselves, and those below 2^-126 have fewer bits.)"""
    for at in (0, 7, 400 // ps - 1):
        s = _case([(1, 400), (1, 900)], 8, 2, hd, ps, seed=12)
        s.vs.fill_(2.0 ** big)
        s.ks.fill_(2.0 ** -9)
        for r in range(2):
            page = int(s.table[r, at])
            s.vs[page] = 2.0 ** -100
            s.v.view(torch.uint8)[page] = 0
            kq = s.q[r].view(2, 4, hd)[:, :1].expand(2, 4, hd).contiguous()
            s.q[r] = kq.reshape(-1)
            s.ks[page] = 2.0 ** -3
            s.k.view(torch.uint8)[page] = (kq[:, 0].float() * (gap * 8 / (1.4427 * hd ** 0.5))).clamp(-448, 448).to(E4M3).view(torch.uint8)[:, None, :].expand(2, ps, hd)
        want = _want(s, None, None if sink is None else torch.full((8,), sink, device=DEV))
        _near(_run(s, sink=sink), want, hd, 2.0 ** -11, 900)
        if gap == 60 and sink is None:
            _near(_run(s, batch=False), want, hd, 0.0, 900)

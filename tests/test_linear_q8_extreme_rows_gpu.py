"""Norms with codes of rows whose squares float32 does not carry: every place of such a row, the filled-up columns among them, against the definition in 64 bits."""
import math

import pytest
import torch

import q8_linear_refs as refs
from arle_b200 import ops
from test_linear_q8_gpu import BF, DEV, F32, _guarded, _near_codes, _rows, _same, _x

pytestmark = pytest.mark.gpu


def _extreme(h, seed):
    """Rows in float32 that are out of the ordinary, each with its name."""
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(h, generator=g)
    base[h // 2] = 1.5
    rows = {"1e20": base * 1e20, "1e16": base * 1e16, "largest": base.clamp(-1, 1) * 3.4e38, "1e-25": base * 1e-25, "denormal": base * 1e-40, "zeros": base * 0.0}
    lone = base * 1e-3
    lone[h // 3] = 2.9e19                                  # one number whose square overflows, or just so
    rows["one large"] = lone
    for name, odd in (("inf", math.inf), ("-inf", -math.inf), ("nan", math.nan)):
        r = base.clone()
        r[h // 3] = odd
        rows[name] = r
    two = base.clone()
    two[0], two[h - 1] = math.inf, -math.inf
    rows["two inf"] = two
    return torch.stack(list(rows.values()))


def _norm64(x, eps, gain):
    x = x.double()
    return x / (x.square().mean(dim=1, keepdim=True) + eps).sqrt() * gain.double()


# a number's product with 1 / sqrt is formed in 64 bits on both sides, in another order: some 2^-50 apart, so that one number in 2^45 could come to the other side of a border
@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("m,h", [(11, 1), (11, 4), (11, 127), (11, 128), (11, 300), (11, 1030), (11, 4096), (11, 5120), (11, 16384), (11, 16500), (300, 516), (300, 1001), (2050, 256), (300, 5120)])
def test_rows_that_float32_does_not_carry(m, h, eps):
    x = _x(m, h, h, 0.5)
    rows = _extreme(h, h)
    at = torch.linspace(0, m - 1, len(rows)).long()
    x[at] = rows
    gain = 1 + 0.3 * torch.randn(h, generator=torch.Generator().manual_seed(m))
    codes, scales = _rows(m, h)
    ops.rmsnorm_q8(x.to(DEV), None, gain.to(DEV), eps, codes[:m], scales[:m])
    _guarded(codes, scales)
    y = _norm64(x, eps, gain)
    mean = x.double().square().mean(dim=1) + eps
    odd = ~((mean > 2.0 ** -90) & (mean < 2.0 ** 100))
    c, s = refs.quantize(y[odd])
    assert odd[at].sum() >= 8
    _same(codes[:m][odd.to(DEV)], c), _same(scales[:m][odd.to(DEV)], s)
    ordinary = (~odd).to(DEV)
    if ordinary.any():
        _near_codes(codes[:m][ordinary], scales[:m][ordinary], y[~odd], (40 + h / 1024) * 2.0 ** -24)
    assert (refs.host(codes[:m])[:, h:] == 0).all()


@pytest.mark.parametrize("place", ["in place", "beside", "nowhere"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,h", [(11, 300), (11, 4096), (11, 1030), (300, 1028), (11, 16500)])
def test_sums_of_such_rows(m, h, dtype, place):
    """With a branch to add: the sum is formed in float32 (it may overflow itself), written where it was asked for, and what it came out as is normed."""
    resid = _x(m, h, h, 0.5)
    rows = _extreme(h, h + 1)
    resid[torch.linspace(0, m - 1, len(rows)).long()] = rows
    delta = (0.1 * _x(m, h, h + 2, 0.5)).to(dtype)
    delta[1] *= 1e19
    delta[2, 0] = 3.3e38
    gain, by, eps = torch.rand(h, generator=torch.Generator().manual_seed(1)) + 0.5, 2.0, 1e-6
    total = resid + by * delta.float()                     # by is a power of two: one rounding, as fma has it
    r = resid.to(DEV)
    out = {"in place": r, "beside": torch.full((m, h), 7.0, device=DEV), "nowhere": None}[place]
    codes, scales = _rows(m, h)
    ops.rmsnorm_q8(r, delta.to(DEV), gain.to(DEV), eps, codes[:m], scales[:m], sum_out=out, delta_scale=by)
    _guarded(codes, scales)
    if out is not None:
        assert torch.equal(out.cpu().nan_to_num(nan=-5.0, posinf=-6.0, neginf=-7.0), total.nan_to_num(nan=-5.0, posinf=-6.0, neginf=-7.0))
    if out is not r:
        assert torch.equal(r.cpu().nan_to_num(nan=-5.0, posinf=-6.0, neginf=-7.0), resid.nan_to_num(nan=-5.0, posinf=-6.0, neginf=-7.0))
    y = _norm64(total, eps, gain)
    mean = total.double().square().mean(dim=1) + eps
    odd = ~((mean > 2.0 ** -90) & (mean < 2.0 ** 100))
    c, s = refs.quantize(y[odd])
    _same(codes[:m][odd.to(DEV)], c), _same(scales[:m][odd.to(DEV)], s)
    assert (refs.host(codes[:m])[:, h:] == 0).all()
    if (~odd).any():
        _near_codes(codes[:m][(~odd).to(DEV)], scales[:m][(~odd).to(DEV)], y[~odd], (40 + h / 1024) * 2.0 ** -24)

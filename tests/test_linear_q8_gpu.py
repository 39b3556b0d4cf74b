"""The linear layers in 8 bits on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

import q8_linear_refs as refs
from arle_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E8M0 = refs.E4M3, refs.E8M0
BF, F32 = torch.bfloat16, torch.float32


def _rows(m, k):
    """Buffers for rows in 8 bits with a guard row behind them that must stay as it is."""
    w = ops.q8_width(k)
    codes = torch.full((m + 1, w), 0x55, dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.full((m + 1, w // 128), 0x33, dtype=torch.uint8, device=DEV).view(E8M0)
    return codes, scales


def _guarded(codes, scales):
    assert (codes.view(torch.uint8)[-1] == 0x55).all() and (scales.view(torch.uint8)[-1] == 0x33).all()


def _same(got, want):
    got = refs.host(got)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def _x(m, k, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(m, k, generator=g) * torch.exp(spread * torch.randn(m, 1, generator=g)) * torch.exp(0.7 * torch.randn(k, generator=g))


# ------------------------------------------------------------------ codes: everything in front of the rounding is exact, so equality is the tolerance
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (2, 129), (7, 256), (5, 264), (1, 4096), (33, 777), (64, 1000), (300, 128)])
def test_quantize(m, k, dtype):
    x = _x(m, k, m * 1000 + k).to(dtype)
    codes, scales = _rows(m, k)
    ops.quantize_q8(x.to(DEV), codes[:m], scales[:m])
    c, s = refs.quantize(x.double())
    _same(codes[:m], c), _same(scales[:m], s), _guarded(codes, scales)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("offset,stride", [(0, 520), (1, 521), (8, 528), (3, 1024)])
def test_quantize_columns_of_a_wider_buffer(offset, stride, dtype):
    wide = _x(9, stride, offset + stride).to(dtype)
    x = wide[:, offset: offset + 512]
    codes, scales = _rows(9, 512)
    ops.quantize_q8(wide.to(DEV)[:, offset: offset + 512], codes[:9], scales[:9])
    c, s = refs.quantize(x.double())
    _same(codes[:9], c), _same(scales[:9], s)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_borders(dtype):
    """Zeros, the ends of a scale's range, ties, maxima at 448 times a power of two and one step around it, numbers that are not finite."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    step = torch.finfo(dtype).eps
    groups = [torch.zeros(128), torch.full((128,), -0.0), torch.full((128,), big), torch.full((128,), small), torch.linspace(-448, 448, 128),
              torch.arange(128) * 2.0 ** -10, torch.arange(128) * 0.5 + 0.25]
    for most in (448.0, 448.0 * (1 + step), 448.0 * (1 - step / 2), 7.0, 2.0 ** -130, 448.0 * 2.0 ** 119, 448.0 * 2.0 ** -100):
        groups.append(torch.linspace(-1, 1, 128) * most)
    for odd in (math.inf, -math.inf, math.nan):
        g = torch.linspace(-3, 3, 128)
        g[5] = odd
        groups += [g, torch.full((128,), odd)]
    x = torch.stack(groups).to(dtype)
    x = torch.cat([x, x.flip(0)], dim=1)
    for shape in (x, x.reshape(1, -1)):
        codes, scales = _rows(*shape.shape)
        m = shape.shape[0]
        ops.quantize_q8(shape.to(DEV), codes[:m], scales[:m])
        c, s = refs.quantize(shape.double())
        _same(codes[:m], c), _same(scales[:m], s), _guarded(codes, scales)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (127, 129), (129, 127), (300, 520), (64, 1031), (257, 256), (1, 4096)])
def test_quantize_weight(n, k, dtype):
    w = (_x(n, k, n + k, 0.5) * 0.02).to(dtype)
    if n > 100:
        w[3, 0], w[17, k // 2], w[90, k - 1] = math.inf, math.nan, -math.inf
        w[: min(n, 128), : 0 if k < 256 else 128] = 0.0
    codes = torch.full((n + 1, ops.q8_width(k)), 0x55, dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.empty((-(-n // 128), -(-k // 128)), device=DEV)
    q = ops.quantize_weight_q8(w.to(DEV), codes[:n], scales)
    c, s = refs.quantize_weight(w.double())
    _same(q.codes, c), _same(q.scales, s)
    assert (codes.view(torch.uint8)[-1] == 0x55).all()


def test_quantize_weight_of_strided_rows():
    w = _x(200, 400, 5).to(BF)
    for cut in (slice(0, 256), slice(1, 257), slice(8, 391)):
        part = w.to(DEV)[:, cut]
        n, k = part.shape
        q = ops.quantize_weight_q8(part, torch.empty((n, ops.q8_width(k)), dtype=E4M3, device=DEV), torch.empty((2, -(-k // 128)), device=DEV))
        c, s = refs.quantize_weight(w[:, cut].double())
        _same(q.codes, c), _same(q.scales, s)


# ------------------------------------------------------------------ rounding of numbers that are known up to a relative error
def _near_codes(codes, scales, y, rel):
    """Rows whose numbers are y up to a relative error ``rel`` each: a group's scale is that of a maximum within ``rel`` of y's, and a value is off by half a
    step of e4m3 (2^-4 of the number, 2^-10 of the scale below 2^-6) beside that error."""
    c, s = refs.host(codes), refs.host(scales)
    m, kb = s.shape
    full = torch.zeros(m, kb * 128, dtype=torch.float64)
    full[:, : y.shape[1]] = y
    most = full.view(m, kb, 128).abs().amax(dim=2)
    assert ((s == refs.scale_of(most * (1 - rel))) | (s == refs.scale_of(most * (1 + rel)))).all()
    got, step = refs.values(c, s), s.repeat_interleave(128, dim=1)
    assert ((got - full).abs() <= (1 + rel) * torch.maximum(full.abs() * 2.0 ** -4, step * 2.0 ** -10) + rel * full.abs()).all()


@pytest.mark.parametrize("dtype", [BF, F32, None])
@pytest.mark.parametrize("m,h", [(1, 1), (1, 128), (3, 127), (5, 1000), (8, 4096), (2, 5120), (3, 1030), (300, 256), (2, 16384), (2, 16500), (1, 20000), (2050, 128), (2048, 1000), (2600, 516), (2100, 1280)])
def test_rmsnorm(m, h, dtype):
    g = torch.Generator().manual_seed(m + h)
    resid, gain = _x(m, h, h, 1.0), 1 + 0.3 * torch.randn(h, generator=g)
    delta = _x(m, h, h + 1, 1.0).to(dtype) if dtype is not None else None
    eps, by = 1e-6, 0.37
    x = resid.double() + (by * delta.double() if delta is not None else 0.0)
    y = x / (x.square().mean(dim=1, keepdim=True) + eps).sqrt() * gain.double()
    codes, scales = _rows(m, h)
    total = torch.full((m + 1, h), 7.0, device=DEV)
    r = resid.to(DEV)
    # the sum is one rounding of a product and a sum (fma), by in float32 itself; the norm: h rounded additions in a tree of at most 16 + h / 1024 deep, squares,
    # the mean, eps, root, quotient, and two products: (30 + h / 1024) half steps, halved by the root for the sum's part; the sum's own error again
    rel = (40 + h / 1024) * 2.0 ** -24
    ops.rmsnorm_q8(r, delta.to(DEV) if delta is not None else None, gain.to(DEV), eps, codes[:m], scales[:m], sum_out=total[:m], delta_scale=by)
    terms = resid.double().abs() + (by * delta.double().abs() if delta is not None else 0.0)
    assert ((total[:m].double().cpu() - x).abs() <= 2.0 ** -23 * terms).all() and (total[m] == 7.0).all()
    x32 = total[:m].double().cpu()          # what the sum came out as is what is normed
    y = x32 / (x32.square().mean(dim=1, keepdim=True) + eps).sqrt() * gain.double()
    _near_codes(codes[:m], scales[:m], y, rel), _guarded(codes, scales)
    again, sagain = _rows(m, h)
    ops.rmsnorm_q8(r, delta.to(DEV) if delta is not None else None, gain.to(DEV), eps, again[:m], sagain[:m], sum_out=r, delta_scale=by)     # in place
    assert torch.equal(r, total[:m]) and torch.equal(again.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(sagain.view(torch.uint8), scales.view(torch.uint8))


def _beside_borders(h):
    """A row and gains whose norm lies within 2^-25 of borders between two codes (of itself), on either side: whole numbers, whose squares' sums float32 holds, so that
    the mean is exact and the numbers in 64 bits are known to 2^-50."""
    g = torch.Generator().manual_seed(h)
    v = torch.randint(1, 256, (h,), generator=g).float()
    border = (torch.randint(8, 16, (h,), generator=g) + 0.5) / 8 * 2.0 ** torch.randint(0, 8, (h,), generator=g)
    border[::128] = 400.0                                   # every group's largest: its scale is 1
    root = v.double().square().mean().sqrt()
    gain = (border.double() * root / v.double()).float()
    return v, gain, v.double() * gain.double() / root, border.double()


@pytest.mark.parametrize("m,h", [(1, 4096), (1, 128), (300, 4096), (300, 1028), (2, 1030), (1, 16384), (3, 16400)])
def test_rmsnorm_beside_borders_between_codes(m, h):
    """A number is rounded once, to its code: rounded to float32 before, four in ten of these would go to the wrong side of the border.  The kernels' factor and
    products are good to 2^-43 (pairs of float32 numbers): numbers that are nearer than 2^-40 to the border do not count."""
    v, gain, y, border = _beside_borders(h)
    codes, scales = _rows(m, h)
    ops.rmsnorm_q8(v.expand(m, h).contiguous().to(DEV), None, gain.to(DEV), 0.0, codes[:m], scales[:m])
    c, s = refs.host(codes[:m]), refs.host(scales[:m])
    want, ws = refs.quantize(y[None])
    sure = ((y - border).abs() > 2.0 ** -40 * border) | (border == 400.0)
    assert sure.double().mean() > 0.99 and (s == ws).all()
    assert (c[:, :h] == want[:, :h])[:, sure].all()
    once, _ = refs.quantize(y[None].float().double())
    assert h < 1000 or (once[:, :h] != want[:, :h]).sum() > h / 10          # (the row tells the two apart)


def test_rmsnorm_rows_at_odd_places():
    """Rows and sums that do not start on 16-byte boundaries take the kernel that reads number by number: the same codes."""
    h = 516
    resid, delta, gain = _x(6, h, 1).to(DEV), _x(6, h, 2).to(DEV), torch.rand(h, device=DEV) + 0.5
    want, swant = _rows(6, h)
    ops.rmsnorm_q8(resid, delta, gain, 1e-5, want[:6], swant[:6])
    odd = [torch.empty(t.numel() + 1, device=DEV)[1:].view(t.shape).copy_(t) for t in (resid, delta, gain)]
    got, sgot = _rows(6, h)
    ops.rmsnorm_q8(*odd, 1e-5, got[:6], sgot[:6])
    x = resid.double().cpu() + delta.double().cpu()
    y = x / (x.square().mean(dim=1, keepdim=True) + 1e-5).sqrt() * gain.double().cpu()
    for c, s in ((want, swant), (got, sgot)):
        _near_codes(c[:6], s[:6], y, 60 * 2.0 ** -24)


def test_rmsnorm_of_a_row_that_is_not_finite():
    resid = _x(3, 300, 3)
    resid[1, 7] = math.inf
    codes, scales = _rows(3, 300)
    ops.rmsnorm_q8(resid.to(DEV), None, torch.ones(300, device=DEV), 1e-6, codes[:3], scales[:3])
    c = refs.host(codes[:3])
    assert c[1, 7].isnan() and c[[0, 2]].isfinite().all()


# ------------------------------------------------------------------ products
def _operands(m, n, k, seed, powers=False):
    g = torch.Generator().manual_seed(seed)
    codes, scales = _rows(m, k)
    ops.quantize_q8(_x(m, k, seed).to(DEV), codes[:m], scales[:m])
    w = 0.02 * torch.randn(n, k, generator=g)
    q = ops.quantize_weight_q8(w.to(DEV), torch.empty((n, ops.q8_width(k)), dtype=E4M3, device=DEV), torch.empty((-(-n // 128), -(-k // 128)), device=DEV))
    if not powers:          # any positive scale is allowed
        q.scales.mul_((0.5 + torch.rand(q.scales.shape, generator=g)).to(DEV))
    return codes[:m], scales[:m], q


def _product(x, sx, q):
    return refs.product(refs.host(x), refs.host(sx), refs.host(q.codes), refs.host(q.scales))


def _close(out, want, size, kb, dtype):
    """A block's sum of 128 exact products, added up in float32 in any order: (128 - 1) half steps of the terms' magnitudes; the scales' product and the
    sum over kb blocks one each; the store's rounding."""
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    bound = (127 + kb + 2) * 2.0 ** -24 * size
    got = out.double().cpu()
    bad = (got - want).abs() > bound + half * (want.abs() + bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / (bound + half * want.abs())).max()):.3g} times the bound"


ROWS = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 500, 513]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(384, 640)])
def test_product_rows(m, n, k):
    x, sx, q = _operands(m, n, k, m)
    want, size = _product(x, sx, q)
    for dtype in (BF, F32):
        out = torch.full((m + 1, n), 3.0, dtype=dtype, device=DEV)
        ops.gemm_q8(x, sx, q, out[:m])
        _close(out[:m], want, size, q.shape[1] // 128, dtype)
        assert (out[m] == 3.0).all()


@pytest.mark.parametrize("m", [1, 5, 20, 70, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 128), (16, 100), (15, 300), (17, 128), (128, 129), (130, 2000), (257, 512), (1000, 777), (2049, 256), (4097, 130), (100, 9000)])
def test_product_sizes(m, n, k):
    x, sx, q = _operands(m, n, k, m + n + k)
    want, size = _product(x, sx, q)
    wide = torch.full((m, n + 3), 3.0, dtype=BF, device=DEV)
    for out in (torch.empty((m, n), device=DEV), wide[:, :n], torch.empty((m, n), dtype=BF, device=DEV), wide[:, 1: n + 1]):
        out.fill_(3.0)
        ops.gemm_q8(x, sx, q, out)
        _close(out, want, size, q.shape[1] // 128, out.dtype)
    assert (wide[:, n + 1:] == 3.0).all()


@pytest.mark.parametrize("m", [1, 8, 24, 64, 128, 300, 1024])
def test_product_is_the_same_every_time(m):
    x, sx, q = _operands(m, 1536, 2048, m)
    outs = [torch.empty((m, 1536), device=DEV) for _ in range(4)]
    for o in outs:
        ops.gemm_q8(x, sx, q, o)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("m", [1, 8, 24, 64, 128, 300])
def test_product_of_extreme_codes(m):
    """Largest codes beside smallest ones in one block, with both signs: the sums cancel down to the smallest products."""
    g = torch.Generator().manual_seed(m)
    n, k = 256, 384
    xc = torch.where(torch.rand(m, k, generator=g) < 0.5, 448.0, 2.0 ** -9) * torch.where(torch.rand(m, k, generator=g) < 0.5, 1.0, -1.0)
    wc = torch.where(torch.rand(n, k, generator=g) < 0.5, 448.0, 2.0 ** -9) * torch.where(torch.rand(n, k, generator=g) < 0.5, 1.0, -1.0)
    sx = torch.exp2(torch.randint(-40, 40, (m, 3), generator=g).float())
    sw = torch.exp2(torch.randint(-20, 20, (2, 3), generator=g).float()) * (1 + torch.rand(2, 3, generator=g))
    x, s, q = xc.to(E4M3).to(DEV), sx.to(E8M0).to(DEV), ops.Q8Weight(wc.to(E4M3).to(DEV), sw.to(DEV))
    out = torch.empty((m, n), device=DEV)
    ops.gemm_q8(x, s, q, out)
    want, size = _product(x, s, q)
    _close(out, want, size, 3, F32)


@pytest.mark.parametrize("m", [1, 8, 24, 64, 128, 300])
def test_product_with_nan(m):
    """A row or a weight's row that holds a NaN gives NaN in its own row or column, and nowhere else."""
    x, sx, q = _operands(m, 300, 512, 11)
    clean = torch.empty((m, 300), device=DEV)
    ops.gemm_q8(x, sx, q, clean)
    x.view(torch.uint8)[m // 2, 77] = 0x7f
    q.codes.view(torch.uint8)[123, 400] = 0xff
    out = torch.empty((m, 300), device=DEV)
    ops.gemm_q8(x, sx, q, out)
    bad = torch.zeros((m, 300), dtype=torch.bool, device=DEV)
    bad[m // 2], bad[:, 123] = True, True
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m", [1, 8, 17, 64, 128, 130, 300, 600])
@pytest.mark.parametrize("i,k", [(128, 128), (100, 300), (384, 640), (1000, 520)])
def test_gated(m, i, k, activation):
    x, sx, gate = _operands(m, i, k, m + i)
    _, _, up = _operands(1, i, k, m + i + 1)
    gate.scales.mul_(20.0)
    w = ops.pack_gate_up_q8(gate, up)
    (gs, gsize), (us, usize) = _product(x, sx, gate), _product(x, sx, up)
    codes, scales = _rows(m, i)
    scratch = torch.empty((m, w.shape[0]), device=DEV)
    ops.gemm_act_mul_q8(x, sx, w, scratch, codes[:m], scales[:m], activation=activation)
    _guarded(codes, scales)
    # the sums' errors as for the product; the gate's slope is at most 1.13 for both, its own arithmetic takes fewer than 16 half steps (and tanh's 2)
    e = (127 + k / 128 + 3) * 2.0 ** -24
    want = refs.act(gs, activation) * us
    off = 1.13 * e * gsize * us.abs() + (refs.act(gs, activation).abs() + e * gsize) * e * usize + 32 * 2.0 ** -24 * (want.abs() + gs.abs() * us.abs() * 2.0 ** -2)
    c, s = refs.host(codes[:m]), refs.host(scales[:m])
    kb = s.shape[1]
    full, err = (torch.zeros(m, kb * 128, dtype=torch.float64) for _ in range(2))
    full[:, :i], err[:, :i] = want, off
    lo = refs.scale_of((full.abs() - err).clamp(min=0.0).view(m, kb, 128).amax(dim=2))
    hi = refs.scale_of((full.abs() + err).view(m, kb, 128).amax(dim=2))
    assert ((s >= lo) & (s <= hi)).all()
    got, step = refs.values(c, s), s.repeat_interleave(128, dim=1)
    assert ((got - full).abs() <= err + torch.maximum((full.abs() + err) * 2.0 ** -4, step * 2.0 ** -10)).all()
    assert (c[:, i:] == 0).all()


@pytest.mark.parametrize("m", [1, 9, 70, 300])
def test_together_as_a_feed_forward(m):
    """Norm, gated product and the last product in a row, captured into a graph and replayed on new numbers, against the same in 64 bits rounded where the
    operators round."""
    h, i = 512, 700
    g = torch.Generator().manual_seed(m)
    ws = [ops.quantize_weight_q8((0.05 * torch.randn(*shape, generator=g)).to(DEV), torch.empty((shape[0], ops.q8_width(shape[1])), dtype=E4M3, device=DEV),
                                 torch.empty((-(-shape[0] // 128), -(-shape[1] // 128)), device=DEV)) for shape in ((i, h), (i, h), (h, i))]
    packed = ops.pack_gate_up_q8(ws[0], ws[1])
    resid, delta, gain = torch.zeros((m, h), device=DEV), torch.zeros((m, h), dtype=BF, device=DEV), torch.rand(h, device=DEV) + 0.5
    (a, sa), (b, sb) = _rows(m, h), _rows(m, i)
    sums, out = torch.empty((m, packed.shape[0]), device=DEV), torch.empty((m, h), dtype=BF, device=DEV)

    def step():
        ops.rmsnorm_q8(resid, delta, gain, 1e-6, a[:m], sa[:m], sum_out=resid)
        ops.gemm_act_mul_q8(a[:m], sa[:m], packed, sums, b[:m], sb[:m])
        ops.gemm_q8(b[:m], sb[:m], ws[2], out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        new, d = _x(m, h, seed, 0.5), _x(m, h, seed + 7, 0.5).to(BF)
        resid.copy_(new), delta.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(out)
        keep = out.clone()
        resid.copy_(new)
        step()
        assert torch.equal(out, keep)
        x = new.double() + d.double()
        y = x / (x.square().mean(dim=1, keepdim=True) + 1e-6).sqrt() * gain.double().cpu()
        c, s = refs.quantize(y)
        gs, us = (refs.product(c, s, refs.host(q.codes), refs.host(q.scales))[0] for q in ws[:2])
        c, s = refs.quantize(refs.act(gs, "silu") * us)
        want, _ = refs.product(c, s, refs.host(ws[2].codes), refs.host(ws[2].scales))
        got = keep.double().cpu()
        # a number next to a border between two codes may fall on either side (2^-3 of itself), which is rare: the result as a whole is near
        assert float((got - want).norm() / want.norm()) < 2.0 ** -8 + 2.0 ** -7
    del eager

"""The 8-bit cache's store on the GPU, against its definition in 64 bits.  Scales are powers of two and codes are rounded once from numbers that
float32 holds exactly, so equality is the tolerance."""
import math

import pytest
import torch

import q8_refs as refs
from arle_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _state(g, pages, nkv, ps, hd, vd):
    """A cache that was written before: random codes (no NaN), scales that are powers of two."""
    caches = []
    for w in (hd, vd):
        x = torch.randn(pages, nkv, ps, w, generator=g) * 100
        caches.append(x.clamp(-448, 448).to(E4M3).to(DEV))
    scales = [torch.exp2(torch.randint(-12, 3, (pages, nkv), generator=g).float()).to(DEV) for _ in range(2)]
    return caches, scales


def _check(x, slots, caches, scales, call, nkv):
    """Runs ``call`` on the caches and compares keys and values with the definition."""
    want = []
    for y, c, s in zip(x, caches, scales):
        c64, s64 = c.float().double().cpu(), s.double().cpu()
        refs.store(y.double().cpu().view(y.shape[0], nkv, -1), slots, c64, s64)
        want.append((c64, s64))
    call()
    for (c64, s64), c, s in zip(want, caches, scales):
        assert torch.equal(s.double().cpu(), s64)
        got = c.float().double().cpu()
        assert torch.equal(got.isnan(), c64.isnan()) and torch.equal(got.nan_to_num(), c64.nan_to_num())


def _slots(g, starts, lens, ps, pages):
    order = torch.randperm(pages, generator=g).tolist()
    slots, at = [], 0
    for s, n in zip(starts, lens):
        have = order[at: at + math.ceil((s + n) / ps)]
        at += len(have)
        slots += [have[p // ps] * ps + p % ps for p in range(s, s + n)]
    return slots


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,hd,vd,ps,starts,lens", [
    (8, 128, 128, 16, [0], [1]),
    (8, 128, 128, 16, [5, 15, 16, 0, 31], [1, 1, 1, 1, 1]),
    (2, 128, 128, 16, [3, 0, 40], [30, 16, 1]),
    (2, 64, 64, 64, [10, 64, 0], [130, 1, 200]),
    (1, 128, 128, 16, [7], [601]),                    # more than 512 tokens: runs are looked for among four tokens at a time
    (2, 80, 48, 48, [9, 0, 3], [700, 1, 50]),
    (3, 33, 33, 8, [3, 8], [21, 2]),
    (1, 6, 256, 4, [1, 2, 3], [9, 1, 1]),
    (1, 256, 256, 100, [50, 1], [301, 70]),
    (2, 64, 64, 1, [3], [5]),
])
def test_store(dtype, nkv, hd, vd, ps, starts, lens):
    g = torch.Generator().manual_seed(hd + ps)
    pages = sum(math.ceil((s + n) / ps) for s, n in zip(starts, lens)) + 3
    caches, scales = _state(g, pages, nkv, ps, hd, vd)
    slots = _slots(g, starts, lens, ps, pages)
    T = len(slots)
    # columns of a wider row, as a packed projection has them
    wide = (torch.randn(T, 7 + nkv * (hd + vd), generator=g) * torch.exp(2 * torch.randn(T, 1, generator=g))).to(dtype).to(DEV)
    for first in (0, 7):
        k, v = wide[:, first: first + nkv * hd], wide[:, first + nkv * hd: first + nkv * (hd + vd)]
        m = torch.tensor(slots, dtype=torch.int32, device=DEV)
        _check((k, v), slots, caches, scales, lambda: ops.store_q8(k, v, m, *caches, *scales, nkv, hd, ps, vd=vd), nkv)


def test_one_token_at_a_time_the_scale_grows():
    g, nkv, hd, ps = torch.Generator().manual_seed(0), 2, 128, 16
    caches, scales = _state(g, 3, nkv, ps, hd, hd)
    for i in range(40):
        x = [(torch.randn(1, nkv * hd, generator=g) * 2.0 ** (i % 16 - 9)).bfloat16().to(DEV) for _ in range(2)]
        slot = [(2 - i // 16) * 16 + i % 16]
        m = torch.tensor(slot, dtype=torch.int32, device=DEV)
        _check(x, slot, caches, scales, lambda: ops.store_q8(*x, m, *caches, *scales, nkv, hd, ps), nkv)


@pytest.mark.parametrize("most", [0.0, 1e-45, 2.0 ** -95, 2.0 ** -92 * 1.75, 2.0 ** -92 * 1.7500001, 448.0, 448.5, 1e30, 3.38e38, math.inf, math.nan])
def test_numbers_at_the_borders(most):
    g, nkv, hd, ps = torch.Generator().manual_seed(1), 1, 64, 16
    caches, scales = _state(g, 2, nkv, ps, hd, hd)
    k = (torch.rand(20, hd, generator=g) - 0.5).double() * 2 * (most if math.isfinite(most) else 3.0)
    k[5, 7], k[18, 60], k[18, 61] = most, -most, most / 2
    k = k.float().to(DEV)
    v = k.flip(0).contiguous()
    slots = list(range(16, 32)) + [0, 1, 2, 3]
    m = torch.tensor(slots, dtype=torch.int32, device=DEV)
    _check((k, v), slots, caches, scales, lambda: ops.store_q8(k, v, m, *caches, *scales, nkv, hd, ps), nkv)


def test_places_that_are_not_stored():
    g, nkv, hd, ps = torch.Generator().manual_seed(2), 2, 128, 16
    caches, scales = _state(g, 4, nkv, ps, hd, hd)
    x = [torch.randn(9, nkv * hd, generator=g).to(DEV) for _ in range(2)]
    slots = [-1, 0, 1, -1, -5, 63, 64, 1 << 30, 32]
    m = torch.tensor(slots, dtype=torch.int32, device=DEV)
    _check(x, slots, caches, scales, lambda: ops.store_q8(*x, m, *caches, *scales, nkv, hd, ps), nkv)
    before = [c.view(torch.uint8).clone() for c in caches]
    none = torch.full((9,), -1, dtype=torch.int32, device=DEV)
    ops.store_q8(*x, none, *caches, *scales, nkv, hd, ps)
    ops.store_q8(x[0][:0], x[1][:0], none[:0], *caches, *scales, nkv, hd, ps)
    assert all(torch.equal(a, c.view(torch.uint8)) for a, c in zip(before, caches))


def test_captured_and_on_another_stream():
    g, nkv, hd, ps = torch.Generator().manual_seed(3), 8, 128, 16
    caches, scales = _state(g, 40, nkv, ps, hd, hd)
    slots = _slots(g, [3, 20, 15], [1, 40, 2], ps, 40)
    m = torch.tensor(slots, dtype=torch.int32, device=DEV)
    x = [torch.randn(len(slots), nkv * hd, generator=g).bfloat16().to(DEV) for _ in range(2)]
    call = lambda: ops.store_q8(*x, m, *caches, *scales, nkv, hd, ps)      # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        for y in x:
            y.copy_(torch.randn(y.shape, generator=g) * 2.0 ** i)
        _check(x, slots, caches, scales, graph.replay, nkv)
    side = torch.cuda.Stream()
    for y in x:
        y.copy_(torch.randn(y.shape, generator=g) * 30)

    def aside():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)

    _check(x, slots, caches, scales, aside, nkv)

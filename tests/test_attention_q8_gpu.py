"""Attention over the 8-bit cache against its definition in 64 bits.

Tolerances, with A = sum p |v| of a number and S the largest |score|: the result's rounding, eps/2 relative.  Scores: products of a bfloat16 number and a
code are exact in float32, their sums and the factors behind them are off by at most (hd + 4) 2^-24 relative to the sum of magnitudes, which the tests'
random numbers keep below 16 times S + 1; a score that is off by d changes a weight by d, and the normalised result by at most 2 d A; exp2 and its argument
add 2^-21 (S + 1).  Weights that are rounded for the product with the values: 2^-11 A (float16) in the decode kernel, 2^-8 A (bfloat16) in the prompt
kernels.  Float32 sums over n keys: n 2^-24 A."""
import math
from types import SimpleNamespace

import pytest
import torch

import q8_refs as refs
from arle_b200 import ops
from arle_b200.engine.batch import Workspace

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def _case(rows, nq, nkv, hd, ps, dtype=BF, vd=None, seed=0, spread=3, fill=0x7f):
    """rows: (queries, keys after the step).  Places of the cache that no row holds carry NaN, pages that no row holds NaN scales too."""
    vd = vd or hd
    g = torch.Generator().manual_seed(seed + hd + ps + nq)
    kvs = [kv for _, kv in rows]
    held = [max(0, math.ceil(kv / ps)) for kv in kvs]
    pages = sum(held) + 4
    order, width = torch.randperm(pages, generator=g).int(), max(held + [1])
    table = torch.full((len(rows), width), -1, dtype=torch.int32)
    k, v = (torch.full((pages, nkv, ps, w), fill, dtype=torch.uint8) for w in (hd, vd))
    ks, vs = (torch.full((pages, nkv), math.nan) for _ in range(2))
    at = 0
    for r, kv in enumerate(kvs):
        table[r, : held[r]] = order[at: at + held[r]]
        at += held[r]
        for j in range(held[r]):
            n = min(ps, kv - j * ps)
            p = int(table[r, j])
            for c, s, base in ((k, ks, -6), (v, vs, -7)):
                c[p, :, :n] = (torch.randn(nkv, n, c.shape[3], generator=g) * 60).clamp(-448, 448).to(E4M3).view(torch.uint8)
                s[p] = torch.exp2((torch.randint(-spread, spread + 1, (nkv,), generator=g) / 2).floor() + base) if c is k else torch.exp2(
                    torch.randint(-spread, spread + 1, (nkv,), generator=g).float() + base)
    indptr = [0]
    for n, _ in rows:
        indptr.append(indptr[-1] + n)
    T = indptr[-1]
    positions = [kv - n + i for n, kv in rows for i in range(n)]
    row_of = [r for r, (n, _) in enumerate(rows) for _ in range(n)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)      # noqa: E731
    s = SimpleNamespace(rows=rows, nq=nq, nkv=nkv, hd=hd, vd=vd, ps=ps, scale=hd ** -0.5, indptr=indptr, kvs=kvs, table=table, T=T)
    s.k, s.v, s.ks, s.vs = k.to(DEV).view(E4M3), v.to(DEV).view(E4M3), ks.to(DEV), vs.to(DEV)
    s.q = torch.randn(T, nq * hd, generator=g).to(dtype).to(DEV)
    s.positions, s.row_of, s.bt = i32(positions), i32(row_of), table.to(DEV)
    lens = [n for n, _ in rows]
    s.batch = SimpleNamespace(q_indptr=i32(indptr), kv_lens=i32(kvs), q_lens=lens, kv_lens_host=kvs, num_rows=len(rows), max_q_len=max(lens), max_kv_len=max(kvs),
                              num_single=sum(n == 1 for n in lens), ws=Workspace(DEV), memo={})
    return s


def _run(s, window=None, sink=None, batch=True):
    out = torch.full((s.T, s.nq * s.vd), 7.0, dtype=s.q.dtype, device=DEV)
    ops.paged_attention_q8(s.q, out, s.k, s.v, s.ks, s.vs, s.positions, s.row_of, s.bt, s.nq, s.nkv, s.hd, s.ps, s.scale, window,
                           batch=s.batch if batch else None, vd=s.vd, sink=sink)
    return out


def _want(s, window=None, sink=None):
    return refs.attention(s.q, s.k.float(), s.v.float(), s.ks, s.vs, s.indptr, s.kvs, s.table, s.nq, s.nkv, s.scale, window, sink)


def _near(out, want, hd, weights, keys):
    ref, size, big = want
    eps = torch.finfo(out.dtype).eps / 2
    d = 16 * (big + 1) * (hd + 4) * 2.0 ** -24 + (big + 1) * 2.0 ** -21
    tol = eps * ref.abs() * 1.01 + size * (weights * 1.01 + 2 * d + keys * 2.0 ** -24) + 1e-30
    off = (out.double() - ref).abs()
    assert out.isfinite().all()
    assert (off <= tol).all(), float((off / tol).max())


DECODE = [[(1, 1)], [(1, 1000)], [(1, 16), (1, 17), (1, 0), (1, 63), (1, 64), (1, 65), (1, 2)], [(1, 300 + 37 * i) for i in range(20)]]


@pytest.mark.parametrize("rows", DECODE, ids=["one", "1000", "edges", "twenty"])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 2), (16, 8), (16, 2), (9, 1), (16, 1)])
@pytest.mark.parametrize("hd,ps", [(128, 16), (64, 64), (128, 12), (64, 5), (128, 48), (128, 1)])
def test_decoded_tokens(rows, nq, nkv, hd, ps):
    s = _case(rows, nq, nkv, hd, ps)
    want = _want(s)
    _near(_run(s), want, hd, 2.0 ** -11, max(s.kvs))
    assert torch.equal(_run(s), _run(s))                       # pieces are joined in the order of keys
    assert not s.batch.ws.get_zeroed("attn_q8_counters", (len(rows) * nkv,), torch.int32).any()
    _near(_run(s, batch=False), want, hd, 0.0, max(s.kvs))


@pytest.mark.parametrize("window", [1, 16, 100, 1000])
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("hd,ps", [(128, 16), (64, 20)])
def test_window_and_sinks(window, sink, hd, ps):
    s = _case([(1, 1), (1, 99), (1, 100), (1, 101), (1, 0), (1, 777), (1, 2100)], 8, 4, hd, ps, seed=4)
    for r, kv in enumerate(s.kvs):                             # pages that the window has passed are given back
        s.table[r, : max(0, kv - window) // ps] = -1
    s.bt = s.table.to(DEV)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(5)).to(DEV) * 3 if sink else None
    want = _want(s, window, sinks)
    _near(_run(s, window, sinks), want, hd, 2.0 ** -11, window)
    _near(_run(s, window, sinks, batch=False), want, hd, 0.0, window)


def test_a_row_without_keys_gets_zeros():
    s = _case([(1, 0), (1, 70), (1, 0)], 8, 2, 128, 16)
    for sink in (None, 0.5):
        for batch in (True, False):
            out = _run(s, sink=sink, batch=batch)
            assert not out[0].any() and not out[2].any() and out[1].any()


@pytest.mark.parametrize("hd", [64, 128])
def test_scales_and_queries_of_all_sizes(hd):
    """Values whose scales lie up to 2^80 apart, and queries from 2^-60 to 2^40: powers of two are taken out of both."""
    s = _case([(1, 900), (1, 33)], 8, 2, hd, 16, spread=40)
    s.ks = torch.full_like(s.ks, 2.0 ** -6)
    want = _want(s)
    _near(_run(s), want, hd, 2.0 ** -11, 900)
    for up in (-60, 40):
        s.q, s.ks = (s.q.double() * 2.0 ** up).to(BF), s.ks * 2.0 ** -up
        _near(_run(s), want, hd, 2.0 ** -11, 900)
        s.q, s.ks = (s.q.double() * 2.0 ** -up).to(BF), s.ks * 2.0 ** up
    s.q[:, :hd] = 0
    _near(_run(s), _want(s), hd, 2.0 ** -11, 900)


@pytest.mark.parametrize("hd,ps", [(64, 16), (128, 16), (128, 12)])
@pytest.mark.parametrize("big", [13, 60])
def test_small_values_that_carry_the_result(hd, ps, big):
    """The keys with all the weight lie in a page whose values are 2^-27 and less, other pages' values are 2^13 or 2^60 times larger; in front and behind."""
    for at in (0, 7, 24):
        s = _case([(1, 400)], 8, 2, hd, ps, seed=11)
        s.vs.fill_(2.0 ** (big - 27))
        page = int(s.table[0, at])
        s.vs[page] = 2.0 ** -27
        # keys of that page along the first query of each kv head, and the queries of a group alike: scores some 300 above the others'
        kq = s.q.view(2, 4, hd)[:, :1].expand(2, 4, hd).contiguous()
        s.q.copy_(kq.reshape(1, -1))
        s.ks.fill_(2.0 ** -9)
        s.ks[page] = 2.0 ** -1
        s.k.view(torch.uint8)[page] = (kq[:, 0].float() * 50).clamp(-448, 448).to(E4M3).view(torch.uint8)[:, None, :].expand(2, ps, hd)
        want = _want(s)
        assert float(want[0].abs().max()) < 2.0 ** -10
        _near(_run(s), want, hd, 2.0 ** -11, 400)
        _near(_run(s, batch=False), want, hd, 0.0, 400)


@pytest.mark.parametrize("where", ["key", "value", "query"])
def test_nan_and_infinity_stay_with_those_who_see_them(where):
    s = _case([(1, 200), (1, 300), (1, 100)], 8, 2, 128, 16)
    clean = _run(s, 50)
    page = int(s.table[1, (300 - 20) // 16])
    before = int(s.table[0, 2])                                # passed by the window
    if where == "query":
        s.q[1, 3] = math.inf
    else:
        cache = s.k if where == "key" else s.v
        for p in (page, before):
            cache.view(torch.uint8)[p, 0, 3, 5] = 0x7f
    out = _run(s, 50)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert out[1].isnan().any() and torch.equal(out[1, 4 * 128:], clean[1, 4 * 128:])


PORTIONS = [[(70, 70)], [(300, 700)], [(5, 90), (1, 400), (129, 129), (1, 1), (2, 2), (64, 1000)], [(33, 33), (1, 0), (300, 301)]]


@pytest.mark.parametrize("rows", PORTIONS, ids=["70", "300", "mixed", "three"])
@pytest.mark.parametrize("hd,ps", [(128, 16), (64, 64), (128, 12)])
@pytest.mark.parametrize("window,sink", [(None, False), (40, False), (256, True)])
@pytest.mark.parametrize("by_tokens", [True, False], ids=["by tokens", "expanded"])
def test_portions(rows, hd, ps, window, sink, by_tokens, monkeypatch):
    monkeypatch.setattr(ops, "_by_tokens_q8", lambda *a: by_tokens)
    s = _case(rows, 8, 2, hd, ps, seed=7)
    if window:
        for r, (n, kv) in enumerate(rows):
            s.table[r, : max(0, kv - n - window + 1) // ps] = -1
        s.bt = s.table.to(DEV)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(5)).to(DEV) if sink else None
    want = _want(s, window, sinks)
    out = _run(s, window, sinks)
    _near(out, want, hd, 2.0 ** -11 if by_tokens else 2.0 ** -8, max(s.kvs))
    _near(_run(s, window, sinks, batch=False), want, hd, 0.0, max(s.kvs))
    assert torch.equal(_run(s, window, sinks), out)
    monkeypatch.setattr(ops, "Q8_EXPAND_BYTES", 1)             # every row by itself: in how many parts its keys are summed goes by the rows that run together
    _near(_run(s, window, sinks), want, hd, 2.0 ** -8, max(s.kvs))
    ops.check_errors(DEV)


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 16, 18])
@pytest.mark.parametrize("rows,window", [([(300, 2100)], None), ([(300, 2100)], 200), ([(257, 257), (1, 900), (2, 700), (600, 1290)], None), ([(2, 2), (130, 130)], 40)])
def test_portions_in_parts(splits, rows, window, monkeypatch):
    """The prompt kernel's key tiles in any number of parts, more than there are tiles among them."""
    s = _case(rows, 8, 2, 128, 16, seed=9)
    monkeypatch.setattr(ops, "prompt_splits_q8", lambda *a: splits)
    monkeypatch.setattr(ops, "_by_tokens_q8", lambda *a: False)
    for sinks in (None, torch.randn(8, generator=torch.Generator().manual_seed(5)).to(DEV)):
        out = _run(s, window, sinks)
        _near(out, _want(s, window, sinks), 128, 2.0 ** -8, max(s.kvs))
        assert torch.equal(_run(s, window, sinks), out)
    ops.check_errors(DEV)


@pytest.mark.parametrize("dtype,hd,vd,nq,nkv,ps", [(torch.float32, 128, 128, 8, 2, 16), (torch.float32, 33, 33, 3, 3, 7), (BF, 80, 80, 4, 1, 16), (BF, 128, 64, 4, 2, 16),
                                                   (BF, 256, 256, 2, 1, 32), (torch.float32, 6, 256, 2, 2, 3), (BF, 128, 128, 34, 2, 16)])
def test_the_general_kernel(dtype, hd, vd, nq, nkv, ps):
    s = _case([(1, 1), (40, 300), (1, 517), (0, 20), (3, 3)], nq, nkv, hd, ps, dtype=dtype, vd=vd)
    for window in (None, 30):
        _near(_run(s, window), _want(s, window), hd, 0.0, 517)


def test_the_plain_kernel_set_and_columns_of_a_wider_row():
    s = _case([(1, 400), (20, 77)], 8, 2, 128, 16)
    wide = torch.zeros(s.T, 8 * 128 + 4 * 128, dtype=BF, device=DEV)
    wide[:, : 8 * 128] = s.q
    s.q = wide[:, : 8 * 128]
    want = _want(s)
    _near(_run(s), want, 128, 2.0 ** -8, 400)
    with ops.use_kernel_set("plain"):
        assert torch.equal(_run(s), _run(s, batch=False))
    s.q = torch.cat([wide[:, :1], wide], dim=1)[:, 1: 1 + 8 * 128]      # rows that are not 16-byte aligned
    _near(_run(s), want, 128, 0.0, 400)


@pytest.mark.parametrize("rows", [[(1, 70), (1, 300)], [(40, 70), (1, 300)]])
def test_no_window(rows):
    s = _case(rows, 8, 2, 128, 16)
    for batch in (True, False):
        all_keys = _run(s, None, batch=batch)
        for window in (0, -5, 10 ** 6):
            assert torch.equal(_run(s, window, batch=batch), all_keys)


@pytest.mark.parametrize("rows", [[(1, 70), (1, 300)], [(3, 70), (1, 300)], [(200, 1500), (1, 300)]], ids=["decoded", "few", "many"])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_rows_behind_the_last_token_are_left_alone(rows, dtype):
    """A padded batch: queries without a request, whose positions and rows are not numbers that anything may be read by."""
    s = _case(rows, 8, 8, 128, 16, dtype=dtype)
    want, pad = _want(s), torch.full((5,), 2 ** 30, dtype=torch.int32, device=DEV)
    s.q, s.positions, s.row_of = torch.cat([s.q, s.q[:1].expand(5, -1)]), torch.cat([s.positions, pad]), torch.cat([s.row_of, pad])
    real, s.T = s.T, s.T + 5
    out = _run(s)
    assert (out[real:] == 7.0).all()
    _near(out[:real], want, 128, 2.0 ** -8, 1500)


def test_an_empty_step(monkeypatch):
    """What step_tables leaves of a step that is not in order: no row has queries or keys, no page is there; nothing is read, in whatever form."""
    for dtype, by_tokens in ((BF, True), (BF, False), (torch.float32, False)):
        monkeypatch.setattr(ops, "_by_tokens_q8", lambda *a, x=by_tokens: x)
        s = _case([(30, 300), (1, 70)], 8, 2, 128, 16, dtype=dtype)
        for x in (s.batch.q_indptr, s.batch.kv_lens, s.positions, s.row_of):
            x.zero_()
        s.bt.fill_(-1)
        _run(s)
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    """Caches of more than 2^32 codes: the pages of a request at their end, for the store, the decoded tokens, portions, and the general kernel."""
    nkv, hd, ps, rows = 8, 128, 16, [(1, 700), (200, 1100), (1, 33)]
    small = _case(rows, 16, nkv, hd, ps)
    pages = 2 ** 32 // (nkv * hd * ps) + 200
    shift = pages - small.k.shape[0]
    s = _case(rows, 16, nkv, hd, ps)
    big = {}
    for n in ("k", "v"):
        big[n] = torch.empty((pages, nkv, ps, hd), dtype=torch.uint8, device=DEV)
        big[n][shift:] = getattr(small, n).view(torch.uint8)
        setattr(s, n, big[n].view(E4M3))
    for n in ("ks", "vs"):
        x = torch.full((pages, nkv), math.nan, device=DEV)
        x[shift:] = getattr(small, n)
        setattr(s, n, x)
    s.bt = torch.where(s.bt >= 0, s.bt + shift, s.bt)
    for batch in (True, False):
        assert torch.equal(_run(s, batch=batch), _run(small, batch=batch))
    x = [torch.randn(40, nkv * hd, generator=torch.Generator().manual_seed(i)).to(DEV) for i in range(2)]
    for c, to in ((small, 0), (s, shift)):
        m = torch.arange(40, dtype=torch.int32, device=DEV) + (to + 2) * ps + 5
        ops.store_q8(*x, m, c.k, c.v, c.ks, c.vs, nkv, hd, ps)
    assert torch.equal(big["k"][shift:], small.k.view(torch.uint8)) and torch.equal(big["v"][shift:], small.v.view(torch.uint8))
    assert torch.equal(s.ks[shift:].nan_to_num(), small.ks.nan_to_num())


def test_a_batch_of_other_types():
    s = _case([(1, 70)], 8, 2, 128, 16)
    s.batch.kv_lens = s.batch.kv_lens.long()
    with pytest.raises(ops.KernelError, match="int32"):
        _run(s)


def test_tensors_of_another_device():
    s = _case([(1, 70)], 8, 2, 128, 16)
    s.ks = s.ks.cpu()
    with pytest.raises(ops.KernelError, match="cpu"):
        _run(s)


def test_a_captured_step_with_portions():
    """The queries and codes change between replays, the lengths stay; decoded tokens run beside the prompt kernel, its parts are joined behind them."""
    s = _case([(70, 800), (1, 700), (300, 301), (1, 1)], 8, 2, 128, 16, seed=3)
    out = torch.empty(s.T, s.nq * s.hd, dtype=BF, device=DEV)

    def call():
        ops.paged_attention_q8(s.q, out, s.k, s.v, s.ks, s.vs, s.positions, s.row_of, s.bt, s.nq, s.nkv, s.hd, s.ps, s.scale, None, batch=s.batch)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(3):
        s.q.copy_(torch.randn(s.q.shape, generator=torch.Generator().manual_seed(step)))
        s.ks *= 2
        graph.replay()
        _near(out, _want(s), 128, 2.0 ** -8, 800)
    ops.check_errors(DEV)


def test_captured_steps_that_share_their_scratch():
    """Two graphs over one workspace, replayed in turn while lengths, queries and codes change."""
    a, b = _case([(1, 700), (1, 90)], 16, 2, 128, 16, seed=1), _case([(1, 200)] * 9, 16, 2, 128, 16, seed=2)
    b.batch.ws = a.batch.ws
    runs = []
    for s in (b, a):
        s.out = torch.empty(s.T, s.nq * s.hd, dtype=BF, device=DEV)
        call = lambda s=s: ops.paged_attention_q8(s.q, s.out, s.k, s.v, s.ks, s.vs, s.positions, s.row_of, s.bt, s.nq, s.nkv, s.hd, s.ps, s.scale, None,      # noqa: E731
                                                  batch=s.batch)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        a.batch.ws.frozen = True
        with torch.cuda.graph(graph):
            call()
        a.batch.ws.frozen = False
        runs.append((s, graph))
    for step in range(3):
        for s, graph in runs:
            s.q.copy_(torch.randn(s.q.shape, generator=torch.Generator().manual_seed(step)))
            s.kvs = [kv - 1 for kv in s.kvs]
            s.batch.kv_lens.copy_(torch.tensor(s.kvs, dtype=torch.int32))
        for s, graph in runs + runs:
            graph.replay()
        for s, _ in runs:
            _near(s.out, _want(s), 128, 2.0 ** -11, max(s.kvs))

"""Every kernel of the 8-bit products with every number of parts, whatever the sizes would choose, and what they share: shared workspaces of captured graphs, streams."""
import subprocess
import sys
import threading

import pytest
import torch

import q8_linear_refs as refs
from arle_b200 import ops
from test_linear_q8_gpu import BF, DEV, E4M3, E8M0, F32, _close, _operands, _product, _rows, _x

pytestmark = pytest.mark.gpu

ROUTES = [("few", p) for p in range(1, 9)] + [("split", p) for p in range(1, 9)] + [("split2", p) for p in range(1, 9)] + [("pair", 1), ("rows", 1)]


@pytest.fixture
def route(monkeypatch):
    def choose(kind, parts):
        monkeypatch.setattr(ops, "_q8_route", lambda M, N, kb, device: (kind, min(parts, kb), 0.0))

    return choose


@pytest.mark.parametrize("kind,parts", ROUTES)
@pytest.mark.parametrize("m", [1, 15, 16, 17, 32, 33, 61, 64, 65, 127, 128, 130, 257])
def test_every_kernel(kind, parts, m, route):
    if kind == "few" and (m > 64 or (m > 32 and parts in (5, 7))):
        pytest.skip("up to 64 rows; five and seven parts up to 32")
    for n, k in ((300, 1200), (129, 8 * 128)):
        x, sx, q = _operands(m, n, k, m + parts)
        want, size = _product(x, sx, q)
        route(kind, parts)
        for dtype in (BF, F32):
            out = torch.full((m + 1, n), 3.0, dtype=dtype, device=DEV)
            ops.gemm_q8(x, sx, q, out[:m])
            _close(out[:m], want, size, q.shape[1] // 128, dtype)
            assert (out[m] == 3.0).all()
        again = torch.empty((m, n), device=DEV)
        ops.gemm_q8(x, sx, q, again)
        assert torch.equal(again, out[:m])          # the parts are added up in their order
    ops.check_errors(DEV)


@pytest.mark.parametrize("kind,parts", [("few", 4), ("few", 1), ("split", 3), ("split2", 2), ("pair", 1)])
def test_long_k_turns_the_rings_over(kind, parts, route):
    m = 40
    x, sx, q = _operands(m, 260, 128 * 131, 3)
    want, size = _product(x, sx, q)
    route(kind, parts)
    out = torch.empty((m, 260), device=DEV)
    ops.gemm_q8(x, sx, q, out)
    _close(out, want, size, 131, F32)


@pytest.mark.parametrize("m", [2, 40, 150, 700])
def test_chains_of_products_that_start_early(m):
    """A row's codes, products and their codes again, forty links without a wait between them: a kernel that starts beside the one in front of it must not read what
    that one is still writing, nor write what it is still reading."""
    h = 384
    w = [_operands(1, h, h, 50 + i)[2] for i in range(3)]
    for q in w:
        q.scales.mul_(10.0)
    x = _x(m, h, 9, 0.5).to(DEV)
    (c, s), y = _rows(m, h), torch.empty((m, h), device=DEV)

    def chain(wait):
        ops.quantize_q8(x, c[:m], s[:m])
        for i in range(40):
            ops.gemm_q8(c[:m], s[:m], w[i % 3], y)
            if wait:
                torch.cuda.synchronize()
            ops.quantize_q8(y, c[:m], s[:m])
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return y.clone()

    want = chain(True)
    assert want.isfinite().all() and torch.equal(chain(False), want)


@pytest.mark.parametrize("m", [3, 50, 200])
def test_weights_that_were_just_made(m):
    """A product right behind the call that makes its weight: the weight is not asked for too early."""
    k, n = 1024, 1536
    g = torch.Generator().manual_seed(m)
    ws = [(0.02 * torch.randn(n, k, generator=g)).to(DEV) for _ in range(2)]
    x, sx, _ = _operands(m, 128, k, m)
    q = ops.Q8Weight(torch.empty((n, k), dtype=E4M3, device=DEV), torch.empty((n // 128, k // 128), device=DEV))
    want = []
    for w in ws:
        ops.quantize_weight_q8(w, q.codes, q.scales)
        torch.cuda.synchronize()
        want.append(torch.empty((m, n), device=DEV))
        ops.gemm_q8(x, sx, q, want[-1])
        torch.cuda.synchronize()
    outs = [torch.empty((m, n), device=DEV) for _ in range(20)]
    for i, out in enumerate(outs):
        ops.quantize_weight_q8(ws[i % 2], q.codes, q.scales)
        ops.gemm_q8(x, sx, q, out)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(outs))


@pytest.mark.parametrize("m", [4, 50, 150, 400])
def test_two_streams_at_once(m):
    """The same weight on two streams, with nothing shared besides: no kernel keeps anything between calls."""
    x, sx, q = _operands(m, 1000, 2048, m)
    y, sy, _ = _operands(m, 128, 2048, m + 1)
    want = []
    for c, s in ((x, sx), (y, sy)):
        want.append(torch.empty((m, 1000), device=DEV))
        ops.gemm_q8(c, s, q, want[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty((m, 1000), device=DEV) for _ in range(10)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(10):
        for j, (c, s) in enumerate(((x, sx), (y, sy))):
            with torch.cuda.stream(streams[j]):
                ops.gemm_q8(c, s, q, outs[j][i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[j]) for j in range(2) for o in outs[j])


def test_two_captured_graphs_with_the_same_buffers():
    """Two graphs that write the same scratch and results, replayed in turn and each after the other."""
    m, k, i = 20, 512, 640
    x, sx, gate = _operands(m, i, k, 1)
    packed = [ops.pack_gate_up_q8(_operands(1, i, k, 10 + j)[2], _operands(1, i, k, 20 + j)[2]) for j in range(2)]
    sums, (c, s) = torch.empty((m, packed[0].shape[0]), device=DEV), _rows(m, i)
    want, graphs = [], []
    for w in packed:
        ops.gemm_act_mul_q8(x, sx, w, sums, c[:m], s[:m])
        torch.cuda.synchronize()
        want.append((c.view(torch.uint8).clone(), s.view(torch.uint8).clone()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.gemm_act_mul_q8(x, sx, w, sums, c[:m], s[:m])
        graphs.append(graph)
    for j in (0, 1, 1, 0, 0, 1):
        graphs[j].replay()
        torch.cuda.synchronize()
        assert torch.equal(c.view(torch.uint8), want[j][0]) and torch.equal(s.view(torch.uint8), want[j][1])


def test_no_rows_and_one_number():
    x, sx, q = _operands(5, 300, 256, 1)
    ops.gemm_q8(x[:0], sx[:0], q, torch.empty((0, 300), device=DEV))
    ops.quantize_q8(torch.empty((0, 5), device=DEV), *[t[:0] for t in _rows(1, 5)])
    ops.rmsnorm_q8(torch.empty((0, 5), device=DEV), None, torch.ones(5, device=DEV), 1e-6, *[t[:0] for t in _rows(1, 5)])
    empty = ops.Q8Weight(torch.empty((0, 256), dtype=E4M3, device=DEV), torch.empty((0, 2), device=DEV))
    ops.gemm_q8(x, sx, empty, torch.empty((5, 0), device=DEV))
    packed = ops.pack_gate_up_q8(q, q)
    ops.gemm_act_mul_q8(x[:0], sx[:0], packed, None if not ops.gate_needs_sums_q8(0, packed) else torch.empty((0, packed.shape[0]), device=DEV),
                        *[t[:0] for t in _rows(1, 300)])


def test_scratch_that_is_missing():
    x, sx, q = _operands(3, 300, 256, 1)
    packed = ops.pack_gate_up_q8(q, q)
    assert ops.gate_needs_sums_q8(3, packed)
    with pytest.raises(ops.KernelError, match="gate_up"):
        ops.gemm_act_mul_q8(x, sx, packed, None, *[t[:3] for t in _rows(3, 300)])


def test_the_plain_kernel_set_takes_the_general_kernels():
    for m in (3, 40, 200):
        x, sx, q = _operands(m, 200, 300, m)
        want, size = _product(x, sx, q)
        out = torch.empty((m, 200), device=DEV)
        with ops.use_kernel_set("plain"):
            ops.gemm_q8(x, sx, q, out)
            packed = ops.pack_gate_up_q8(q, q)
            assert ops.gate_needs_sums_q8(m, packed)
        _close(out, want, size, 3, F32)


def test_offsets_beyond_32_bits():
    """A weight of more than 2^32 codes, and results of more than 2^31 numbers: rows at their ends."""
    n, k, m = 140_000, 32_768, 9
    codes = torch.zeros((n, k), dtype=torch.uint8, device=DEV)
    codes[-3:] = torch.randint(0, 120, (3, k), dtype=torch.uint8, device=DEV)
    scales = torch.ones((-(-n // 128), k // 128), device=DEV)
    q = ops.Q8Weight(codes.view(E4M3), scales)
    last = ops.Q8Weight(q.codes[-96:].contiguous(), scales[-1:].contiguous())          # 140,000 = 1,093 * 128 + 96
    for rows in (2, m, 70):
        x, sx, _ = _operands(rows, 128, k, rows)
        out = torch.empty((rows, n), device=DEV)
        ops.gemm_q8(x, sx, q, out)
        want, size = _product(x, sx, last)
        _close(out[:, -96:], want, size, k // 128, F32)
        assert (out[:, :-96] == 0).all()
    del codes, q, out
    m, n = 33_000, 70_000
    x, sx, q = _operands(64, n, 128, 5)
    xs, ss = x.view(torch.uint8).repeat(516, 1)[:m].view(E4M3), sx.view(torch.uint8).repeat(516, 1)[:m].view(E8M0)
    out = torch.empty((m, n), dtype=BF, device=DEV)
    ops.gemm_q8(xs, ss, q, out)
    first = torch.empty((64, n), dtype=BF, device=DEV)
    ops.gemm_q8(xs[:64], ss[:64], q, first)
    # both are roundings of sums in other orders of the same 128 products
    assert torch.equal(out[-8:], out[m - 8 - 64 * 10: m - 64 * 10]) and ((out[:64].float() - first.float()).abs() <= 2.0 ** -7 * first.float().abs() + 1e-3).all()


def test_two_threads_at_once():
    """Calls from two threads, a stream each."""
    sizes = ((4, 1000, 2048), (150, 640, 1024))
    made = [_operands(*size, 3) for size in sizes]
    want = []
    for (m, n, _), (x, sx, q) in zip(sizes, made):
        want.append(torch.empty((m, n), device=DEV))
        ops.gemm_q8(x, sx, q, want[-1])
    torch.cuda.synchronize()
    same = [None, None]

    def work(j):
        (m, n, _), (x, sx, q) = sizes[j], made[j]
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [torch.empty((m, n), device=DEV) for _ in range(40)]
            for out in outs:
                ops.gemm_q8(x, sx, q, out)
            torch.cuda.current_stream().synchronize()
            same[j] = all(torch.equal(out, want[j]) for out in outs)

    threads = [threading.Thread(target=work, args=(j,)) for j in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [True, True]


FIRST_CALLS = """
import torch
from arle_b200 import ops
g = torch.Generator().manual_seed(0)
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
q = ops.Q8Weight(torch.randint(0, 100, (512, 1024), dtype=torch.uint8, generator=g).cuda().view(E4M3), torch.ones((4, 8), device="cuda"))
x = torch.randn((300, 1024), generator=g).cuda()
codes, scales = torch.empty((300, 1024), dtype=E4M3, device="cuda"), torch.empty((300, 8), dtype=torch.uint8, device="cuda").view(E8M0)
gc, gs = torch.empty((300, 256), dtype=E4M3, device="cuda"), torch.empty((300, 2), dtype=torch.uint8, device="cuda").view(E8M0)
sums = torch.empty((300, 512), device="cuda")
outs = {m: torch.zeros((m, 512), device="cuda") for m in (1, 20, 130, 300)}
torch.cuda.synchronize()

def calls():
    ops.quantize_q8(x, codes, scales)
    for m, out in outs.items():
        ops.gemm_q8(codes[:m], scales[:m], q, out)
    ops.gemm_act_mul_q8(codes, scales, q, sums, gc, gs)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
graph.replay()
torch.cuda.synchronize()
kept = {m: out.clone() for m, out in outs.items()}
gated = gc.view(torch.uint8).clone()
calls()
torch.cuda.synchronize()
assert all(torch.equal(kept[m], out) and out.abs().max() > 0 for m, out in outs.items()) and torch.equal(gated, gc.view(torch.uint8))
ops.check_errors(x.device)
print("captured")
"""


def test_a_process_whose_first_calls_are_captured():
    """What a kernel's first launch needs (shared memory limits, how many clusters run, the error word) is there or may be had while a graph is captured."""
    from pathlib import Path

    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]

"""A weight whose codes the kernel in front of a product writes, one that lets the product start early."""
import pytest
import torch

from arle_b200 import ops
from test_linear_q8_gpu import DEV, E4M3, E8M0, _operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 3, 8, 20, 50, 100, 200, 400])
@pytest.mark.parametrize("n,k", [(1536, 1024), (4096, 4096), (300, 8192)])
def test_codes_that_a_kernel_has_just_written(m, n, k):
    g = torch.Generator().manual_seed(m)
    ws = [torch.randn(n, k, generator=g).to(DEV) for _ in range(2)]
    x, sx, _ = _operands(m, 128, k, m)
    q = ops.Q8Weight(torch.empty((n, k), dtype=E4M3, device=DEV), torch.ones((-(-n // 128), k // 128), device=DEV))
    row_scales = torch.empty((n, k // 128), dtype=torch.uint8, device=DEV).view(E8M0)
    want = []
    for w in ws:
        ops.quantize_q8(w, q.codes, row_scales)
        torch.cuda.synchronize()
        want.append(torch.empty((m, n), device=DEV))
        ops.gemm_q8(x, sx, q, want[-1])
        torch.cuda.synchronize()
    assert not torch.equal(*want)
    outs = [torch.empty((m, n), device=DEV) for _ in range(20)]

    def step():
        for i, out in enumerate(outs):
            ops.quantize_q8(ws[i % 2], q.codes, row_scales)
            ops.gemm_q8(x, sx, q, out)

    step()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(outs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for out in outs:
        out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(outs))


@pytest.mark.parametrize("kind,parts,m", [("pair", 1, 300), ("pair", 1, 2100), ("split", 3, 300), ("split2", 2, 300), ("few", 4, 60), ("rows", 1, 8)])
def test_chains_with_every_kernel_launched_early(kind, parts, m, monkeypatch):
    """Forty links of codes, product and codes again, all kernels launched programmatically: the same as with a wait behind each."""
    h = 1024
    monkeypatch.setattr(ops, "_q8_route", lambda M, N, kb, device: (kind, parts, 0.0))
    g = torch.Generator().manual_seed(m)
    ws = [_operands(1, h, h, 70 + i)[2] for i in range(3)]
    for q in ws:
        q.scales.mul_(10.0)
    x, y = torch.randn(m, h, generator=g).to(DEV), torch.empty((m, h), device=DEV)
    c, s = torch.empty((m, h), dtype=E4M3, device=DEV), torch.empty((m, h // 128), dtype=torch.uint8, device=DEV).view(E8M0)

    def chain(wait):
        ops.quantize_q8(x, c, s)
        for i in range(40):
            ops.gemm_q8(c, s, ws[i % 3], y)
            if wait:
                torch.cuda.synchronize()
            ops.quantize_q8(y, c, s)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return y.clone()

    want = chain(True)
    ops.set_programmatic_launch(1)
    try:
        got = chain(False)
    finally:
        ops.set_programmatic_launch(0)
    assert want.isfinite().all() and torch.equal(got, want)
    ops.check_errors(DEV)

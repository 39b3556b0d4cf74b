"""What the linear layers in 8 bits refuse, before anything is launched, and how weights are packed."""
import pytest
import torch

import q8_linear_refs as refs
from arle_b200 import ops

BF, F8, E8, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float32


def z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype) if dtype in (F8, E8) else torch.zeros(*shape, dtype=dtype)


def _weight(n=300, k=256):
    return ops.Q8Weight(z(n, k, dtype=F8), z(-(-n // 128), k // 128))


def _quantize(**changed):
    a = dict(x=z(4, 200, dtype=BF), codes=z(4, 256, dtype=F8), scales=z(4, 2, dtype=E8))
    a.update(changed)
    ops.quantize_q8(**a)


def _quantize_weight(**changed):
    a = dict(w=z(300, 200, dtype=BF), codes=z(300, 256, dtype=F8), scales=z(3, 2))
    a.update(changed)
    ops.quantize_weight_q8(**a)


def _norm(**changed):
    a = dict(resid=z(4, 200), delta=z(4, 200, dtype=BF), weight=z(200), eps=1e-6, codes=z(4, 256, dtype=F8), scales=z(4, 2, dtype=E8))
    a.update(changed)
    ops.rmsnorm_q8(**a)


def _product(**changed):
    a = dict(codes=z(4, 256, dtype=F8), scales=z(4, 2, dtype=E8), w=_weight(), out=z(4, 300, dtype=BF))
    a.update(changed)
    ops.gemm_q8(**a)


def _gated(**changed):
    a = dict(codes=z(4, 256, dtype=F8), scales=z(4, 2, dtype=E8), w=_weight(512), gate_up=z(4, 512), out_codes=z(4, 256, dtype=F8), out_scales=z(4, 2, dtype=E8))
    a.update(changed)
    ops.gemm_act_mul_q8(**a)


def _gate(**changed):
    a = dict(gate_up=z(4, 512), codes=z(4, 256, dtype=F8), scales=z(4, 2, dtype=E8))
    a.update(changed)
    ops.act_mul_q8(**a)


ROWS = [dict(codes=z(4, 256, dtype=BF)), dict(codes=z(3, 256, dtype=F8)), dict(codes=z(4, 200, dtype=F8)), dict(codes=z(4, 0, dtype=F8)), dict(codes=z(256, 4, dtype=F8).t()),
        dict(codes=z(4, 512, dtype=F8)[:, :256]), dict(scales=z(4, 2)), dict(scales=z(4, 3, dtype=E8)), dict(scales=z(2, 4, dtype=E8).t()), dict(scales=z(8, dtype=E8)),
        dict(codes=z(4, 384, dtype=F8), scales=z(4, 3, dtype=E8))]


@pytest.mark.parametrize("changed", ROWS + [dict(x=z(4, 200, dtype=torch.float16)), dict(x=z(800, dtype=BF)), dict(x=z(200, 4).t()), dict(x=z(4, 0)), dict(x=z(4, 257)),
                                            dict(x=z(5, 200))])
def test_quantize(changed):
    with pytest.raises(ops.KernelError):
        _quantize(**changed)


@pytest.mark.parametrize("changed", [dict(w=z(300, 200, dtype=torch.float64)), dict(w=z(200, 300).t()), dict(w=z(60000)), dict(w=z(300, 0)), dict(w=z(299, 200)),
                                     dict(codes=z(300, 256, dtype=torch.uint8)), dict(codes=z(300, 384, dtype=F8)), dict(scales=z(3, 2, dtype=BF)), dict(scales=z(2, 2)),
                                     dict(scales=z(2, 3).t())])
def test_quantize_weight(changed):
    with pytest.raises(ops.KernelError):
        _quantize_weight(**changed)


@pytest.mark.parametrize("changed", ROWS + [dict(resid=z(4, 200, dtype=BF)), dict(resid=z(200, 4).t()), dict(resid=z(4, 0)), dict(delta=z(4, 200, dtype=torch.float16)),
                                            dict(delta=z(4, 201)), dict(delta=z(200, 4).t()), dict(weight=z(200, dtype=BF)), dict(weight=z(199)), dict(weight=z(400)[::2]),
                                            dict(sum_out=z(4, 200, dtype=BF)), dict(sum_out=z(4, 201)), dict(sum_out=z(200, 4).t())])
def test_norm(changed):
    with pytest.raises(ops.KernelError):
        _norm(**changed)


@pytest.mark.parametrize("changed", ROWS + [dict(out=z(4, 299)), dict(out=z(3, 300)), dict(out=z(300, 4).t()), dict(out=z(1, 300).expand(4, 300)), dict(out=z(4, 300, dtype=torch.float16)), dict(w=_weight(300, 384))])
def test_product(changed):
    with pytest.raises(ops.KernelError):
        _product(**changed)


@pytest.mark.parametrize("changed", ROWS + [dict(w=_weight(300)), dict(w=_weight(384)), dict(gate_up=z(4, 512, dtype=BF)), dict(gate_up=z(4, 300)), dict(gate_up=z(512, 4).t()),
                                            dict(out_codes=z(4, 384, dtype=F8)), dict(out_scales=z(4, 2)), dict(activation="relu")])
def test_gated(changed):
    with pytest.raises(ops.KernelError):
        _gated(**changed)


@pytest.mark.parametrize("changed", ROWS + [dict(gate_up=z(4, 512, dtype=BF)), dict(gate_up=z(4, 511)), dict(gate_up=z(512, 4).t()), dict(activation="relu")])
def test_gate(changed):
    with pytest.raises(ops.KernelError):
        _gate(**changed)


@pytest.mark.parametrize("codes,scales", [(z(300, 256), z(3, 2)), (z(300, 200, dtype=F8), z(3, 2)), (z(300, 0, dtype=F8), z(3, 0)), (z(256, dtype=F8), z(1, 2)),
                                          (z(256, 300, dtype=F8).t(), z(3, 2)), (z(300, 256, dtype=F8), z(3, 2, dtype=BF)), (z(300, 256, dtype=F8), z(2, 2)),
                                          (z(300, 256, dtype=F8), z(2, 3).t()), (z(76832, dtype=F8)[3: 76803].view(300, 256), z(3, 2))])
def test_weight(codes, scales):
    with pytest.raises(ops.KernelError):
        ops.Q8Weight(codes, scales)


def test_tensors_of_the_cpu():
    for call in (_quantize, _quantize_weight, _norm, _product, _gated, _gate):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


@pytest.mark.parametrize("i,k", [(128, 128), (100, 256), (300, 384)])
def test_pack(i, k):
    """Rows of a packed weight: 128 of the gate, 128 of the other, zeros at the end."""
    g = torch.Generator().manual_seed(i)
    parts = [refs.quantize_weight(torch.randn(i, k, generator=g).double()) for _ in range(2)]
    gate, up = (ops.Q8Weight(c.to(F8), s.float()) for c, s in parts)
    w = ops.pack_gate_up_q8(gate, up)
    nb = -(-i // 128)
    assert tuple(w.shape) == (256 * nb, k)
    full = refs.weight_values(refs.host(w.codes), refs.host(w.scales)).view(nb, 2, 128, k)
    for j, q in enumerate((gate, up)):
        rows = full[:, j].reshape(nb * 128, k)
        assert torch.equal(rows[:i], refs.weight_values(refs.host(q.codes), refs.host(q.scales))) and (rows[i:] == 0).all()
    with pytest.raises(ops.KernelError):
        ops.pack_gate_up_q8(gate, ops.Q8Weight(z(i + 1, k, dtype=F8), z(-(-(i + 1) // 128), k // 128)))


def test_first_rows():
    c, s = refs.quantize_weight(torch.randn(300, 256, generator=torch.Generator().manual_seed(0)).double())
    q = ops.Q8Weight(c.to(F8), s.float())
    for n in (1, 128, 129, 300):
        part = q.first_rows(n)
        assert torch.equal(refs.weight_values(refs.host(part.codes), refs.host(part.scales)), refs.weight_values(c, s)[:n])


def test_widths():
    assert [ops.q8_width(k) for k in (1, 127, 128, 129, 4096)] == [128, 128, 128, 256, 4096]

"""Gates in 8 bits by themselves and in the plain kernel set, and a model in 8 bits on the GPU against one whose matrices and rows were rounded beforehand."""
import math

import pytest
import torch

import q8_linear_refs as refs
from arle_b200 import ops
from arle_b200.engine import ModelRunner, StepEntry
from arle_b200.engine.loading import random_model
from test_linear_q8_gpu import DEV, _guarded, _operands, _product, _rows, _same, _x
from test_weights_q8_engine_gpu import CONFIG

pytestmark = pytest.mark.gpu


def _near(codes, scales, want, off):
    """Codes and scales of numbers that are ``want`` up to ``off`` each: a group's scale is that of a maximum within that, a value is off by half a step of e4m3 beside it."""
    c, s = refs.host(codes), refs.host(scales)
    m, kb = s.shape
    full, err = (torch.zeros(m, kb * 128, dtype=torch.float64) for _ in range(2))
    full[:, : want.shape[1]], err[:, : want.shape[1]] = want, off
    lo = refs.scale_of((full.abs() - err).clamp(min=0.0).view(m, kb, 128).amax(dim=2))
    hi = refs.scale_of((full.abs() + err).view(m, kb, 128).amax(dim=2))
    assert ((s >= lo) & (s <= hi)).all()
    got, step = refs.values(c, s), s.repeat_interleave(128, dim=1)
    assert ((got - full).abs() <= err + torch.maximum((full.abs() + err) * 2.0 ** -4, step * 2.0 ** -10)).all()
    assert (c[:, want.shape[1]:] == 0).all()


def _gate_error(g, u, want):
    """A gate's own arithmetic in float32: fewer than 16 half steps of the result and of a quarter of |g u| (silu's exponential is off by |g| 2^-24 of itself, tanh by two
    steps of one, and a gate that ends near zero is a difference of numbers near |g| / 2)."""
    return 32 * 2.0 ** -24 * (want.abs() + g.abs() * u.abs() * 2.0 ** -2)


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,nb", [(1, 1), (3, 5), (64, 96), (700, 7), (5000, 3)])
def test_gate_of_sums(m, nb, activation):
    g, u = 4.0 * _x(m, nb * 128, m + nb, 0.3), _x(m, nb * 128, m + nb + 1, 1.0)
    sums = torch.stack([g.view(m, nb, 128), u.view(m, nb, 128)], dim=2).reshape(m, -1)
    codes, scales = _rows(m, nb * 128)
    before = ops.launch_count()
    ops.act_mul_q8(sums.to(DEV), codes[:m], scales[:m], activation=activation)
    assert ops.launch_count() == before + 1
    _guarded(codes, scales)
    g, u = g.double(), u.double()
    want = refs.act(g, activation) * u
    _near(codes[:m], scales[:m], want, _gate_error(g, u, want))


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_gate_borders(activation):
    """Gates of either sign from zero to the ends of float32, results that are not finite (they become NaN and do not count), groups with nothing but those."""
    ends = [0.0, -0.0, 1e-30, -1e-30, 1.0, -1.0, 20.0, -20.0, 87.0, -87.0, 88.0, -88.0, 89.0, -89.0, 127.0, -127.0, -200.0, 1e10, -1e10, 1e30, -1e30, 3e38, -3e38]
    g = torch.linspace(-3, 3, 128).repeat(5, 1)
    g[0, : len(ends)] = torch.tensor(ends)
    g[1, 3], g[1, 50], g[1, 127] = math.inf, -math.inf, math.nan
    g[2] = math.nan
    u = torch.ones(5, 128)
    u[3, 7], u[3, 8] = math.nan, math.inf
    u[0] = 1e-8                                            # (so that the largest of the group does not leave the scale's range)
    u[4] = 0.0
    u[4, 5] = -2.0
    codes, scales = _rows(5, 128)
    ops.act_mul_q8(torch.cat([g, u], dim=1).to(DEV), codes[:5], scales[:5], activation=activation)
    _guarded(codes, scales)
    c, s = refs.host(codes[:5]), refs.host(scales[:5])
    odd = ~(g.isfinite() & u.isfinite())
    assert torch.equal(c.isnan(), odd) and s[2, 0] == 2.0 ** refs.LOW
    gd, ud = torch.where(odd, 0.0, g).double(), torch.where(odd, 0.0, u).double()
    want = refs.act(gd, activation).nan_to_num(0.0) * ud
    off = _gate_error(gd, ud, want)
    got, step = refs.values(c.nan_to_num(0.0), s), s.expand(5, 128)
    assert ((got - want).abs() <= off + torch.maximum((want.abs() + off) * 2.0 ** -4, step * 2.0 ** -10)).all()


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,i,k", [(1, 128, 128), (3, 100, 300), (40, 384, 640), (70, 129, 257), (200, 256, 520), (600, 130, 1000)])
def test_gated_product_of_the_plain_set(m, i, k, activation):
    x, sx, gate = _operands(m, i, k, m + i)
    _, _, up = _operands(1, i, k, m + i + 1)
    gate.scales.mul_(20.0)
    w = ops.pack_gate_up_q8(gate, up)
    (gs, gsize), (us, usize) = _product(x, sx, gate), _product(x, sx, up)
    codes, scales = _rows(m, i)
    with ops.use_kernel_set("plain"):
        assert ops.gate_needs_sums_q8(m, w)
        ops.gemm_act_mul_q8(x, sx, w, torch.empty((m, w.shape[0]), device=DEV), codes[:m], scales[:m], activation=activation)
    _guarded(codes, scales)
    # a block's sum and the sum over blocks: (127 + blocks + 3) half steps of the terms' magnitudes; the gate's slope is at most 1.13
    e = (127 + -(-k // 128) + 3) * 2.0 ** -24
    want = refs.act(gs, activation) * us
    off = 1.13 * e * gsize * us.abs() + (refs.act(gs, activation).abs() + e * gsize) * e * usize + _gate_error(gs, us, want)
    _near(codes[:m], scales[:m], want, off)


def test_a_model_s_weights_are_the_rounded_matrices():
    """Codes and scales of every matrix of every layer, packed as the products take them, are those of the wide model's matrices: equal, so that a scale which is wrong in
    one block shows.  (Logits do not show it: an error of 2^-10 moves numbers across borders between codes in the next layer, and a model's kernel sets end hundredths apart.)"""
    model, wide = (random_model(CONFIG, 9, "bfloat16", DEV, sigma=0.05, weight_dtype=w) for w in ("float8_e4m3", "auto"))
    assert len(model.blocks) == 3
    for b, w in zip(model.blocks, wide.blocks):
        for got, want in ((b.mixer.w_qkv, w.mixer.w_qkv), (b.mixer.w_o, w.mixer.w_o), (b.ffn.w_down, w.ffn.w_down)):
            c, s = refs.quantize_weight(want.double().cpu())
            _same(got.codes, c), _same(got.scales, s)
        packed, i = b.ffn.w_gate_up, CONFIG["intermediate_size"]
        for j in (0, 1):
            c, s = refs.quantize_weight(w.ffn.w_gate_up[j::2].double().cpu())
            rows = refs.host(packed.codes).view(-1, 2, 128, packed.shape[1])[:, j].reshape(-1, packed.shape[1])
            assert torch.equal(rows[:i], c) and (rows[i:] == 0).all()
            _same(packed.scales.view(-1, 2, packed.scales.shape[1])[:, j], s)


@pytest.mark.parametrize("kernel_set", ["fast", "plain"])
def test_one_layer_is_that_of_rounded_matrices_and_rows(kernel_set, monkeypatch):
    """A float32 layer in 8 bits beside the ordinary path on the same numbers: matrices rounded beforehand, rows rounded in front of every product.  Sums are of float32
    on both sides, some 2^-20 apart, so one number in 2^15 comes to the other side of a border between two codes.  A row has some 3,100 numbers that are rounded: nine
    rows in ten have none of those and end 2^-16 apart or less; the others differ by what one code is off.  (A wrong scale in a block moves every row.)"""
    config = dict(CONFIG, num_hidden_layers=1)
    model, wide = (random_model(config, 9, "float32", DEV, sigma=0.05, weight_dtype=w) for w in ("float8_e4m3", "auto"))

    def rounded(t, quantize=refs.quantize, values=refs.values):
        return values(*quantize(t.double().cpu()))[:, : t.shape[1]].float().to(DEV)

    def rounded_matrix(w):
        return rounded(w, refs.quantize_weight, refs.weight_values)

    b = wide.blocks[0]
    for part, name in ((b.mixer, "w_qkv"), (b.mixer, "w_o"), (b.ffn, "w_down")):
        setattr(part, name, rounded_matrix(getattr(part, name)))
    g = b.ffn.w_gate_up.float()
    b.ffn.w_gate_up = torch.stack([rounded_matrix(g[0::2]), rounded_matrix(g[1::2])], dim=1).reshape(g.shape).contiguous()
    ids = torch.randint(0, 999, (40,), generator=torch.Generator().manual_seed(2)).tolist()

    def run(m):
        r = ModelRunner(m, 16, 60, 2, 800, DEV, kernel_set=kernel_set)
        out = [r.step([StepEntry("a", ids[a:b], tuple(range(b - a)))]).clone() for a, b in ((0, 20), (20, 21), (21, 40))]
        ops.check_errors(DEV)
        return torch.cat(out).double()

    got = run(model)
    plain, gate, head = ops.gemm, ops.gemm_act_mul, wide.head
    monkeypatch.setattr(ops, "gemm", lambda x, w, out, sink=None, **kw: plain(x if w is head else rounded(x), w, out, sink=sink, **kw))
    monkeypatch.setattr(ops, "gemm_act_mul", lambda x, w, gu, out, activation="silu", **kw: gate(rounded(x), w, gu, out, activation, **kw))
    want = run(wide)
    off = (got - want).norm(dim=1) / want.norm(dim=1)
    assert float(off.median()) < 2.0 ** -16

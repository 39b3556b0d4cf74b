"""What is measured of the linear layers in 8 bits, and their plain forms.

A number is an e4m3 code times a scale: activations have one scale, a power of two, for each row and 128 numbers of k; weights one float32 scale for
each block of 128 x 128.  k is filled up to a multiple of 128 with codes of zero.

``quantize``   a step's activations as codes and scales
``weight``     a weight matrix as codes and scales, once, when a model is loaded
``norm``       the residual sum and the RMSNorm in front of a product, its result as codes and scales
``product``    rows of activations times a weight matrix
``gated``      the first half of a gated feed-forward: both products, silu(gate) * up, the result as codes and scales

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls that a program makes of ``arle_b200.ops``.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
B = 128                        # numbers of a block
E4M3_MOST = 448.0
LOW, HIGH = -100, 119          # exponents that a scale of activations may have
EPS = 1e-6
LARGEST = 4096 * 24576 * 4096  # rows * columns * k of the largest listed case


def listed():
    return [
        # one user's chat: what attention leaves of one token, in front of the output projection of the 8B size; launch latency is all there is
        dict(name="quantize, one token", op="quantize", m=1, k=4096, dtype="bfloat16"),
        # a prompt step of the 32B size in front of the output projection
        dict(name="quantize, 6,001 tokens", op="quantize", m=6001, k=8192, dtype="bfloat16"),
        # loading: the packed gate and up matrices of the 8B size
        dict(name="weight, 24,576 x 4,096", op="weight", n=24576, k=4096, dtype="bfloat16"),
        # loading a small model that is stored in 32 bits, sizes that end inside a block
        dict(name="weight, 1,001 x 777", op="weight", n=1001, k=777, dtype="float32"),
        # a small decode step between two products of the 8B size
        dict(name="norm, 8 tokens", op="norm", m=8, k=4096, dtype="bfloat16"),
        # a prompt step of the 32B size
        dict(name="norm, 5,003 tokens", op="norm", m=5003, k=5120, dtype="bfloat16"),
        # one user's chat: the output projection of the 8B size
        dict(name="product, one token", op="product", m=1, n=4096, k=4096, out="bfloat16"),
        # a server's decode step: the packed query, key and value projections of the 8B size
        dict(name="product, 64 tokens", op="product", m=64, n=6144, k=4096, out="bfloat16"),
        # a short prompt beside decoded tokens: the last product of the feed-forward of the 32B size
        dict(name="product, 333 tokens", op="product", m=333, n=5120, k=25600, out="bfloat16"),
        # a long prompt's portion: the last product of the feed-forward of the 8B size
        dict(name="product, 4,096 tokens", op="product", m=4096, n=4096, k=12288, out="bfloat16"),
        # a small decode step: the feed-forward of the 8B size
        dict(name="gated, 8 tokens", op="gated", m=8, n=12288, k=4096),
        # a long prompt's portion through the same
        dict(name="gated, 4,096 tokens", op="gated", m=4096, n=12288, k=4096),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _width(rng, hi):
    """A layer's width: now and then one that is no multiple of anything."""
    w = _log(rng, 64, hi)
    return w if rng.random() < 0.3 else max(64, w // 64 * 64)


def draw(rng):
    op = rng.choice(["quantize", "weight", "norm", "product", "product", "product", "gated", "gated"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op in ("quantize", "norm"):
        return dict(op=op, m=_log(rng, 1, 5000), k=_width(rng, 5120 if op == "norm" else 8192), dtype=dtype)
    if op == "weight":
        return dict(op=op, n=_width(rng, 16384), k=_width(rng, 4096), dtype=dtype)
    n, k = _width(rng, 12288), _width(rng, 12288)
    m = _log(rng, 1, max(1, min(4096, LARGEST // (2 * n * k))))
    return dict(op=op, m=m, n=n, k=k, out=rng.choice(["bfloat16", "bfloat16", "float32"])) if op == "product" else dict(op=op, m=m, n=n, k=k)


def _blocks(k):
    return -(-k // B)


def work(case):
    k = case["k"]
    size = 4 if "float32" in (case.get("dtype"), case.get("out")) else 2
    if case["op"] == "quantize":
        return {"bytes": case["m"] * (k * (size + 1) + _blocks(k)), "flops": 0}
    if case["op"] == "weight":
        return {"bytes": case["n"] * k * (size + 1) + 4 * _blocks(case["n"]) * _blocks(k), "flops": 0}
    if case["op"] == "norm":
        return {"bytes": case["m"] * (k * (4 + size + 4 + 1) + _blocks(k)) + 4 * k, "flops": 0}
    m, n = case["m"], case["n"]
    rows = m * (k + _blocks(k))
    if case["op"] == "product":
        return {"bytes": rows + n * k + 4 * _blocks(n) * _blocks(k) + m * n * size, "flops": 2 * m * n * k}
    return {"bytes": rows + 2 * (n * k + 4 * _blocks(n) * _blocks(k)) + m * (n + _blocks(n)), "flops": 4 * m * n * k}


# ------------------------------------------------------------------ inputs
def _activations(g, m, k, dtype=torch.float32):
    """Activations as a layer makes them: a few channels are much larger than the others, and tokens differ in size."""
    x = torch.randn((m, k), generator=g, device=DEV)
    x *= torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))
    x *= torch.exp(0.4 * torch.randn((m, 1), generator=g, device=DEV))
    return x.to(dtype)


def _empty_rows(m, k):
    return (torch.empty((m, _blocks(k) * B), dtype=torch.float8_e4m3fn, device=DEV),
            torch.empty((m, _blocks(k)), dtype=torch.float8_e8m0fnu, device=DEV))


def _stored_weight(g, n, k):
    """Codes and scales of a weight as a checkpoint stores them: a scale is the block's largest number / 448."""
    nb, kb = _blocks(n), _blocks(k)
    w = torch.randn((nb * B, kb * B), generator=g, device=DEV)
    w *= 0.02 * torch.exp(0.3 * torch.randn((nb, 1, kb, 1), generator=g, device=DEV)).expand(nb, B, kb, B).reshape(nb * B, kb * B)
    w[n:] = 0.0
    w[:, k:] = 0.0
    blocks = w.view(nb, B, kb, B)
    scale = blocks.abs().amax(dim=(1, 3)) / E4M3_MOST
    codes = (blocks / scale[:, None, :, None]).clamp(-E4M3_MOST, E4M3_MOST).reshape(nb * B, kb * B).to(torch.float8_e4m3fn)
    return codes[:n].contiguous(), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    op, k = case["op"], case["k"]
    if op == "weight":
        n = case["n"]
        w = 0.02 * torch.randn((n, k), generator=g, device=DEV)
        w *= torch.exp(0.5 * torch.randn((n, 1), generator=g, device=DEV))
        return dict(case=case, w=w.to(DTYPES[case["dtype"]]), codes=torch.empty((n, _blocks(k) * B), dtype=torch.float8_e4m3fn, device=DEV),
                    scales=torch.empty((_blocks(n), _blocks(k)), device=DEV))
    m = case["m"]
    if op == "quantize":
        codes, scales = _empty_rows(m, k)
        return dict(case=case, x=_activations(g, m, k, DTYPES[case["dtype"]]), codes=codes, scales=scales)
    if op == "norm":
        codes, scales = _empty_rows(m, k)
        return dict(case=case, resid=4.0 * _activations(g, m, k), delta=_activations(g, m, k, DTYPES[case["dtype"]]),
                    gain=1.0 + 0.2 * torch.randn(k, generator=g, device=DEV), total=torch.empty((m, k), device=DEV), codes=codes, scales=scales)
    x, sx = _quantize_plain(_activations(g, m, k))
    if op == "product":
        w, sw = _stored_weight(g, case["n"], k)
        return dict(case=case, x=x, sx=sx, w=w, sw=sw, out=torch.empty((m, case["n"]), dtype=DTYPES[case["out"]], device=DEV))
    # rows of the packed weight: 128 of the gate, 128 of the up projection, and so on; the last blocks are filled up with zeros
    nb = _blocks(case["n"])
    parts = [_stored_weight(g, case["n"], k) for _ in range(2)]
    fill = nb * B - case["n"]
    both = torch.stack([torch.nn.functional.pad(c.view(torch.uint8), (0, 0, 0, fill)).view(nb, B, -1) for c, _ in parts], dim=1)
    w = both.reshape(2 * nb * B, -1).view(torch.float8_e4m3fn)
    sw = torch.stack([s for _, s in parts], dim=1).reshape(2 * nb, -1).contiguous()
    codes, scales = _empty_rows(m, case["n"])
    return dict(case=case, x=x, sx=sx, w=w, sw=sw, sums=torch.empty((m, 2 * nb * B), device=DEV), codes=codes, scales=scales)


# ------------------------------------------------------------------ plain forms
def _scale_of(most):
    """The smallest power of two s with most / s <= 448 = 1.75 * 2^8 (most = f * 2^e with f in [0.5, 1): 2^(e - 9), doubled where f > 0.875)."""
    f, e = torch.frexp(most)
    e = torch.where(most > 0, e - 9 + (f > 0.875).to(e.dtype), LOW).clamp(LOW, HIGH)
    return torch.ldexp(torch.ones_like(most), e)


def _codes(x, scale):
    return torch.where(torch.isfinite(x), (x / scale).clamp(-E4M3_MOST, E4M3_MOST), math.nan).to(torch.float8_e4m3fn)


def _quantize_plain(y):
    m, k = y.shape
    y = torch.nn.functional.pad(y.float(), (0, -k % B)).view(m, -1, B)
    scale = _scale_of(torch.where(torch.isfinite(y), y.abs(), 0.0).amax(dim=2))
    return _codes(y, scale[:, :, None]).view(m, -1), scale.to(torch.float8_e8m0fnu)


def _weight_plain(w):
    n, k = w.shape
    y = torch.nn.functional.pad(w.float(), (0, -k % B, 0, -n % B)).view(_blocks(n), B, _blocks(k), B)
    scale = _scale_of(torch.where(torch.isfinite(y), y.abs(), 0.0).amax(dim=(1, 3)))
    return _codes(y, scale[:, None, :, None]).view(-1, _blocks(k) * B)[:n], scale


def _norm_plain(resid, delta, gain):
    x = resid + delta.float()
    return x, *_quantize_plain(x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS) * gain)


def _product_plain(x, sx, w, sw):
    m, kb = sx.shape
    rows = (x.float().view(m, kb, B) * sx.float()[:, :, None]).view(m, -1)
    fill = sw.shape[0] * B - w.shape[0]
    full = torch.nn.functional.pad(w.float(), (0, 0, 0, fill)).view(-1, B, kb, B) * sw[:, None, :, None]
    return torch.matmul(rows, full.view(-1, kb * B)[: w.shape[0]].T)


def _gated_plain(x, sx, w, sw):
    sums = _product_plain(x, sx, w, sw).view(x.shape[0], -1, 2, B)
    gate, up = sums[:, :, 0], sums[:, :, 1]
    return _quantize_plain((gate / (1.0 + torch.exp(-gate)) * up).reshape(x.shape[0], -1))


# ------------------------------------------------------------------ a pass
def _handle(s):
    """The weight as a program keeps it, made once when a model is loaded."""
    if "handle" not in s:
        from arle_b200 import ops

        s["handle"] = ops.Q8Weight(s["w"], s["sw"])
    return s["handle"]


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from arle_b200 import ops
    if op == "quantize":
        if own:
            ops.quantize_q8(s["x"], s["codes"], s["scales"])
            return s["codes"], s["scales"]
        return _quantize_plain(s["x"])
    if op == "weight":
        if own:
            ops.quantize_weight_q8(s["w"], s["codes"], s["scales"])
            return s["codes"], s["scales"]
        return _weight_plain(s["w"])
    if op == "norm":
        if own:
            ops.rmsnorm_q8(s["resid"], s["delta"], s["gain"], EPS, s["codes"], s["scales"], sum_out=s["total"])
            return s["total"], s["codes"], s["scales"]
        return _norm_plain(s["resid"], s["delta"], s["gain"])
    if op == "product":
        if own:
            ops.gemm_q8(s["x"], s["sx"], _handle(s), s["out"])
            return s["out"]
        return _product_plain(s["x"], s["sx"], s["w"], s["sw"]).to(s["out"].dtype)
    if own:
        ops.gemm_act_mul_q8(s["x"], s["sx"], _handle(s), s["sums"], s["codes"], s["scales"], activation="silu")
        return s["codes"], s["scales"]
    return _gated_plain(s["x"], s["sx"], s["w"], s["sw"])


# ------------------------------------------------------------------ in 64 bits
def _exact_scale(most):
    """By its definition: the least power of two that carries ``most``, found from a logarithm that may be off by one."""
    near = torch.round(torch.log2((most / E4M3_MOST).clamp(min=2.0 ** -140)))
    scale = torch.exp2((near + 2).clamp(LOW, HIGH))
    for less in (1, 0, -1):
        smaller = torch.exp2((near + less).clamp(LOW, HIGH))
        scale = torch.where(most <= E4M3_MOST * smaller, smaller, scale)
    return scale


def _exact_codes(y, scale):
    """The nearest e4m3 number, ties to the even one: steps of 2^-9 below 2^-6, of an eighth of their power of two above."""
    t = (y / scale).clamp(-E4M3_MOST, E4M3_MOST)
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    step = torch.where(t.abs() >= 16 * step, 2 * step, torch.where(t.abs() < 8 * step, (step / 2).clamp(min=2.0 ** -9), step))
    return torch.round(t / step) * step


def _exact_rows(y):
    m, k = y.shape
    kb = _blocks(k)
    full = torch.zeros((m, kb * B), dtype=torch.float64, device=y.device)
    full[:, :k] = y
    scale = _exact_scale(full.view(m, kb, B).abs().amax(dim=2))
    return _exact_codes(full.view(m, kb, B), scale[:, :, None]).reshape(m, -1), scale


def _exact_sums(s, cut=2048):
    sx, sw = s["sx"].float().double(), s["sw"].double()
    rows = s["x"].float().double() * sx.repeat_interleave(B, dim=1)
    n = s["w"].shape[0]
    out = torch.empty((rows.shape[0], n), dtype=torch.float64, device=rows.device)
    for a in range(0, n, cut):
        b = min(n, a + cut)
        scale = sw[a // B: _blocks(b)].repeat_interleave(B, dim=0)[: b - a].repeat_interleave(B, dim=1)
        out[:, a:b] = rows @ (s["w"][a:b].float().double() * scale).T
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rows(s["x"].double())
    if op == "norm":
        x = s["resid"].double() + s["delta"].double()
        y = x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / case["k"] + EPS) * s["gain"].double()
        return (x, *_exact_rows(y))
    if op == "product":
        return _exact_sums(s)
    if op == "gated":
        sums = _exact_sums(s).reshape(case["m"], -1, 2, B)
        return _exact_rows((sums[:, :, 0] * torch.sigmoid(sums[:, :, 0]) * sums[:, :, 1]).reshape(case["m"], -1))
    n, k = case["n"], case["k"]
    codes = torch.zeros((n, _blocks(k) * B), dtype=torch.float64, device=DEV)
    scales = torch.empty((_blocks(n), _blocks(k)), dtype=torch.float64, device=DEV)
    codes[:, :k] = s["w"].double()
    for i in range(_blocks(n)):
        rows = codes[i * B: (i + 1) * B].view(-1, _blocks(k), B)
        scales[i] = _exact_scale(rows.abs().amax(dim=(0, 2)))
        rows.copy_(_exact_codes(rows, scales[i][None, :, None]))
    return codes, scales

"""The linear layers in 8 bits in 64 bits, by their definitions: codes and scales as float64 values."""
import torch

B, MOST, LOW, HIGH = 128, 448.0, -100, 119
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

# all e4m3 numbers that are not negative, in order: the code is the place
GRID = torch.arange(127, dtype=torch.uint8).view(E4M3).double()


def scale_of(most):
    """The least power of two that carries ``most``, by trying all of them."""
    powers = torch.tensor([2.0 ** e for e in range(LOW, HIGH + 1)], dtype=torch.float64)
    return powers[(most.unsqueeze(-1) > MOST * powers).sum(dim=-1).clamp(max=len(powers) - 1)]


def round_e4m3(t):
    """The nearest of all e4m3 numbers, ties to the even code; NaN stays, what is larger ends at the largest."""
    a = t.abs().clamp(max=MOST)
    hi = torch.searchsorted(GRID, a.nan_to_num(0.0)).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - GRID[lo], GRID[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    v = torch.copysign(GRID[pick], t)
    return torch.where(t.isnan(), torch.nan, v)


def quantize(x):
    """x [M, K] float64 -> (codes' values [M, 128 kb], scales [M, kb])."""
    m, k = x.shape
    kb = -(-k // B)
    full = torch.zeros(m, kb * B, dtype=torch.float64)
    full[:, :k] = x
    full = full.view(m, kb, B)
    s = scale_of(torch.where(full.isfinite(), full.abs(), 0.0).amax(dim=2)) if m else torch.zeros(0, kb, dtype=torch.float64)
    c = round_e4m3(torch.where(full.isfinite(), full, torch.nan) / s[:, :, None])
    return c.view(m, kb * B), s


def quantize_weight(w):
    n, k = w.shape
    nb, kb = -(-n // B), -(-k // B)
    full = torch.zeros(nb * B, kb * B, dtype=torch.float64)
    full[:n, :k] = w
    full = full.view(nb, B, kb, B)
    s = scale_of(torch.where(full.isfinite(), full.abs(), 0.0).amax(dim=(1, 3)))
    c = round_e4m3(torch.where(full.isfinite(), full, torch.nan) / s[:, None, :, None])
    return c.view(nb * B, kb * B)[:n], s


def values(codes, scales):
    """What rows of codes stand for."""
    return codes * scales.repeat_interleave(B, dim=1)


def weight_values(codes, scales):
    return codes * scales.repeat_interleave(B, dim=0)[: codes.shape[0]].repeat_interleave(B, dim=1)


def product(x, sx, w, sw):
    """(the product, the sum of its terms' magnitudes)."""
    a, b = values(x, sx), weight_values(w, sw)
    return a @ b.T, a.abs() @ b.abs().T


def act(g, activation):
    if activation == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)))


def host(t):
    return t.float().double().cpu() if t.dtype in (E4M3, E8M0) else t.double().cpu()

"""Weights that a checkpoint stores in 8 bits: e4m3 codes "<name>" beside float32 (or 16-bit) scales "<name>_scale_inv", one for each block of 128 x 128; a
weight is code * scale.  cklxx/arle reads such pairs for its quantised weights (infer/src/weight_loader.rs); here they are kept as they are by the parts that run on
them and turned into the engine's type by all others.
"""
from __future__ import annotations

import warnings
from typing import Optional, Sequence

import torch

BLOCK = 128
SCALE_SUFFIX = "_scale_inv"


class StoredQ8:
    """A stored matrix [N, K]: ``codes`` float8_e4m3fn [N, K] and ``scales`` float32 [ceil(N / 128), ceil(K / 128)], on the host.  ``to`` gives its numbers
    (bfloat16 where no type is asked for), so a part that knows nothing of codes loads it like any other tensor.  ``dtype`` is what holds them, four bits times a float32
    scale: an engine of 32 bits keeps them as such."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        n, k = codes.shape
        if tuple(scales.shape) != (-(-n // BLOCK), -(-k // BLOCK)):
            raise ValueError(f"scales {tuple(scales.shape)} do not fit codes {tuple(codes.shape)} in blocks of {BLOCK}")
        self.codes, self.scales, self.shape = codes, scales.to(torch.float32), codes.shape
        self.dtype = torch.float32

    def to(self, device=None, dtype=None) -> torch.Tensor:
        codes, scales = self.codes.to(device=device), self.scales.to(device=device)
        n, k = self.shape
        out = torch.empty((n, k), dtype=dtype or torch.bfloat16, device=codes.device)
        for i in range(0, n, 32 * BLOCK):                  # a few blocks of rows at a time: in float32 a matrix is four times its codes
            j = min(n, i + 32 * BLOCK)
            s = scales[i // BLOCK: -(-j // BLOCK)].repeat_interleave(BLOCK, dim=0)[: j - i].repeat_interleave(BLOCK, dim=1)[:, :k]
            out[i:j] = (codes[i:j].to(torch.float32) * s).to(out.dtype)
        return out


def as_tensor(t, dtype: torch.dtype) -> torch.Tensor:
    """A stored tensor as one: codes become the numbers of an engine of this type."""
    return t.to(dtype=dtype) if isinstance(t, StoredQ8) else t


def as_q8_weight(parts: Sequence, device) -> Optional["ops.Q8Weight"]:
    """Stored matrices one under the other as one weight with their own codes and scales; None where that cannot be (one of them is not stored in 8 bits, or ends
    inside a block that the next one would share)."""
    from .. import ops

    if not all(isinstance(p, StoredQ8) for p in parts) or any(p.shape[0] % BLOCK for p in parts[:-1]):
        return None
    n, k = sum(p.shape[0] for p in parts), parts[0].shape[1]
    codes = torch.zeros((n, ops.q8_width(k)), dtype=torch.uint8, device=device)
    at = 0
    for p in parts:
        codes[at: at + p.shape[0], :k] = p.codes.view(torch.uint8).to(device)
        at += p.shape[0]
    return ops.Q8Weight(codes.view(torch.float8_e4m3fn), torch.cat([p.scales for p in parts]).to(device).contiguous())


def q8_weight(matrix) -> "ops.Q8Weight":
    """A matrix on the device as codes and scales."""
    from .. import ops

    n, k = matrix.shape
    codes = torch.empty((n, ops.q8_width(k)), dtype=torch.float8_e4m3fn, device=matrix.device)
    return ops.quantize_weight_q8(matrix, codes, torch.empty((-(-n // ops.Q8_BLOCK), codes.shape[1] // ops.Q8_BLOCK), dtype=torch.float32, device=matrix.device))


def stored_q8_weight(tensors: dict, names: Sequence[str], device) -> "ops.Q8Weight":
    """The named matrices one under the other as codes and scales: a checkpoint's own where one weight can have them, else found from the numbers as they are stored (in
    16 or 32 bits; code * scale in 32), so that these are rounded once."""
    matrices = [tensors[n] for n in names]
    own = as_q8_weight(matrices, device)
    if own is not None:
        return own
    if any(isinstance(m, StoredQ8) for m in matrices):
        warnings.warn(f"{', '.join(names)}: stored in 8 bits, but not all of them, or two would share a block of 128 rows: the codes are found anew")
    wide = torch.bfloat16 if all(m.dtype == torch.bfloat16 for m in matrices) else torch.float32
    return q8_weight(torch.cat([m.to(device=device, dtype=wide) for m in matrices]))

"""Learned codes looked up by number - the discrete sibling of the grids (`tinycudann.Encoding`, `sparsegrid.SparseGrid`), for what a clip is
conditioned on by index rather than by coordinate: frame, clip, shot, token.  No counterpart in the reference.

    out[i] = scale * table[ids[i]]            a negative id is an empty slot (a row of zeros, no gradient)

The gradient is dense, like the grids': dtable[v] = scale * the sum of dout over the positions with id v, added in fp32 in a fixed order
(positions sorted by id; no atomics, bit-reproducible) and written once.  An id >= the number of codes is a mistake: its row is NaN, it has no
gradient, and with NVP_CHECK_IDS=1 the call raises instead (a device synchronisation per call)."""
from __future__ import annotations

import os

import torch
from torch import nn

from . import _lib as L

CHECK_IDS = os.environ.get("NVP_CHECK_IDS", "0") == "1"


def lookup(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, dtype: torch.dtype | None = None) -> torch.Tensor:
    """ids [...] (int64 / int32), table [codes, dim] (fp32 / bf16 / fp16) -> [..., dim] of `dtype` (default: the table's; an fp32 table may be read
    as bf16 or fp16).  Differentiable with respect to the table, whose gradient has the table's type; differentiable once."""
    return L.binding().lookup(ids, table, scale, dtype, CHECK_IDS)


class CodeTable(nn.Module):
    """`n_codes` learned codes of `dim` values: parameter `codes` [n_codes, dim], U(-1e-4, 1e-4) like the grids; forward(ids) = scale * codes[ids]."""

    def __init__(self, n_codes: int, dim: int, scale: float = 1.0, dtype: torch.dtype = torch.float32, out_dtype: torch.dtype | None = None):
        super().__init__()
        if n_codes < 1 or dim < 1:
            raise ValueError("CodeTable needs at least one code of at least one value")
        self.n_codes, self.dim, self.scale, self.out_dtype = n_codes, dim, float(scale), out_dtype
        self.codes = nn.Parameter(torch.empty(n_codes, dim, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self):
        std = 1e-4
        self.codes.data.uniform_(-std, std)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return lookup(ids, self.codes, self.scale, self.out_dtype)

    def extra_repr(self) -> str:
        return f"n_codes={self.n_codes}, dim={self.dim}, scale={self.scale}"

"""Residual stack between learned codes and the modulated SIREN's latent (`modulation.SirenWrapper.forward(coords, latent)`).  No counterpart in the
reference, whose only conditioning step is SirenNet's `x *= mod` (modulation.py:83-92).

One step, with the norms on both sides of a block fused with its gate and residual scale into one kernel per direction:

    u = pre_norm(x, w0)                                   in front of the first block
    h = block(u)
    y, u = gated_residual(x, h, gate, post, next)         y = x + scale * act(gate) * h / rms(h) * post,  u = y / rms(y) * next

rms(v) = sqrt(mean(v^2) + eps) over the last dimension.  Streams (x, h, gate, y, u) share one type, fp32 / bf16 / fp16; the weights are fp32 or of
that type; arithmetic and sums are fp32.  `u` is computed from y before y is rounded."""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L
from .quantize import Linear8

_ACTS = {None: 0, "sigmoid": 1}
MAX_DIM = 8192


def pre_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """x [..., D] -> x / rms(x) * weight, of x's type."""
    return L.binding().pre_norm(x, weight, eps)


def gated_residual(x: torch.Tensor, h: torch.Tensor, gate: torch.Tensor | None, post_weight: torch.Tensor, next_weight: torch.Tensor | None = None, scale: float = 1.0,
                   gate_act: str | None = None, eps: float = 1e-6):
    """x, h [..., D] -> y = x + scale * act(gate) * h / rms(h) * post_weight; with `next_weight` (the norm in front of the next block) the pair
    (y, y / rms(y) * next_weight).  gate: None (1), x's shape, or x's shape with 1 in place of the last leading dimensions (one gate row for all the
    rows below it: [B, 1, D] for x [B, T, D]); gate_act None or 'sigmoid'.  Differentiable (once) with respect to every tensor."""
    act = _ACTS.get(gate_act)
    if act is None:
        raise RuntimeError(f"gated_residual: gate_act must be None or 'sigmoid', got {gate_act!r}")
    out = L.binding().gated_residual(x, h, gate, post_weight, next_weight, scale, act, eps)
    return out[0] if next_weight is None else (out[0], out[1])


class Trunk(nn.Module):
    """`depth` residual blocks of width `dim` (Linear -> LeakyReLU -> Linear, as the Modulator's layers, with a sigmoid gate from the block's input):
    code [..., dim] -> latent [..., dim], normed at the end.  `to_8bit()` gives the copy for 8-bit evaluation (quantize.Linear8 layers)."""

    def __init__(self, dim: int, depth: int, hidden: int | None = None, scale: float | None = None, eps: float = 1e-6):
        super().__init__()
        if dim < 1 or dim > MAX_DIM or depth < 1:
            raise ValueError(f"Trunk needs 1 <= dim <= {MAX_DIM} and at least one block")
        hidden = 4 * dim if hidden is None else hidden
        self.dim, self.depth, self.eps = dim, depth, eps
        self.scale = depth ** -0.5 if scale is None else float(scale)
        self.norms = nn.ParameterList([nn.Parameter(torch.ones(dim)) for _ in range(depth + 1)])          # in front of every block, and the last one
        self.posts = nn.ParameterList([nn.Parameter(torch.ones(dim)) for _ in range(depth)])
        self.ups = nn.ModuleList([nn.Linear(dim, hidden) for _ in range(depth)])
        self.downs = nn.ModuleList([nn.Linear(hidden, dim) for _ in range(depth)])
        self.gates = nn.ModuleList([nn.Linear(dim, dim) for _ in range(depth)])
        self.act = nn.LeakyReLU()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        u = pre_norm(x, self.norms[0], self.eps)
        for k in range(self.depth):
            h = self.downs[k](self.act(self.ups[k](u))).to(x.dtype)                   # (under autocast the linear layers answer in its type)
            x, u = gated_residual(x, h, self.gates[k](u).to(x.dtype), self.posts[k], self.norms[k + 1], self.scale, "sigmoid", self.eps)
        return u

    @torch.no_grad()
    def to_8bit(self) -> "Trunk":
        """A copy whose linear layers are quantize.Linear8 (weights and activations in blocks of 128; inference only).  Needs parameters on a HIP device."""
        other = Trunk.__new__(Trunk)
        nn.Module.__init__(other)
        other.dim, other.depth, other.eps, other.scale = self.dim, self.depth, self.eps, self.scale
        other.norms = nn.ParameterList([nn.Parameter(p.detach().clone(), requires_grad=False) for p in self.norms])
        other.posts = nn.ParameterList([nn.Parameter(p.detach().clone(), requires_grad=False) for p in self.posts])
        for name in ("ups", "downs", "gates"):
            setattr(other, name, nn.ModuleList([Linear8.from_linear(m) for m in getattr(self, name)]))
        other.act = nn.LeakyReLU()
        return other

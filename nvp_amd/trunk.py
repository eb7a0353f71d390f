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
from .functional import GatedResidual
from .quantize import Linear8

_ACTS = {None: 0, "sigmoid": 1}
MAX_DIM = 8192


def _weight(w: torch.Tensor, x: torch.Tensor, what: str) -> None:
    if tuple(w.shape) != (x.shape[-1],) or w.dtype not in (torch.float32, x.dtype):
        raise RuntimeError(f"{what}: expected a weight [{x.shape[-1]}] of float32 or {x.dtype}, got {w.dtype} {tuple(w.shape)}")


def _stream(x: torch.Tensor, what: str) -> None:
    L.stream_type(x, what)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise RuntimeError(f"{what}: expected [..., D] with 1 <= D <= {MAX_DIM}, got {tuple(x.shape)}")


def _eps(eps: float, what: str) -> float:
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError(f"{what}: eps must be finite and not negative, got {eps}")
    return eps


def _gate_rows(x: torch.Tensor, gate: torch.Tensor) -> int:
    """How many rows of D the gate has; row r of x uses gate row r // (rows of x // rows of the gate): the gate's leading dimensions are x's up to
    some point and 1 from there on (dimensions missing on the left count as 1)."""
    lead, got = list(x.shape[:-1]), list(gate.shape[:-1]) if gate.dim() else None
    ok = got is not None and gate.dtype == x.dtype and gate.shape[-1] == x.shape[-1] and len(got) <= len(lead)
    if ok:
        got = [1] * (len(lead) - len(got)) + got
        k = len(got)
        while k and got[k - 1] == 1:
            k -= 1
        ok = got[:k] == lead[:k]
    if not ok:
        raise RuntimeError(f"gated_residual: a gate for x {tuple(x.shape)} ({x.dtype}) has its type and its shape, or 1 in place of the last leading dimensions, "
                           f"got {gate.dtype} {tuple(gate.shape)}")
    return gate.numel() // gate.shape[-1]


def pre_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """x [..., D] -> x / rms(x) * weight, of x's type."""
    _stream(x, "pre_norm")
    _weight(weight, x, "pre_norm")
    return GatedResidual.apply(x, None, None, None, weight, 1, 1.0, 0, _eps(eps, "pre_norm"), torch.is_grad_enabled())[1]


def gated_residual(x: torch.Tensor, h: torch.Tensor, gate: torch.Tensor | None, post_weight: torch.Tensor, next_weight: torch.Tensor | None = None, scale: float = 1.0,
                   gate_act: str | None = None, eps: float = 1e-6):
    """x, h [..., D] -> y = x + scale * act(gate) * h / rms(h) * post_weight; with `next_weight` (the norm in front of the next block) the pair
    (y, y / rms(y) * next_weight).  gate: None (1), x's shape, or x's shape with 1 in place of the last leading dimensions (one gate row for all the
    rows below it: [B, 1, D] for x [B, T, D]); gate_act None or 'sigmoid'.  Differentiable with respect to every tensor."""
    _stream(x, "gated_residual")
    if h.shape != x.shape or h.dtype != x.dtype:
        raise RuntimeError(f"gated_residual: h must be like x ({x.dtype} {tuple(x.shape)}), got {h.dtype} {tuple(h.shape)}")
    _weight(post_weight, x, "gated_residual")
    if next_weight is not None:
        _weight(next_weight, x, "gated_residual")
        if next_weight.dtype != post_weight.dtype:
            raise RuntimeError(f"gated_residual: the two weights must be of one type, got {post_weight.dtype} and {next_weight.dtype}")
    if gate_act not in _ACTS:
        raise RuntimeError(f"gated_residual: gate_act must be None or 'sigmoid', got {gate_act!r}")
    scale = float(scale)
    if scale != scale or scale in (float("inf"), float("-inf")):
        raise RuntimeError(f"gated_residual: scale must be finite, got {scale}")
    gate_rows = _gate_rows(x, gate) if gate is not None else 1
    y, u = GatedResidual.apply(x, h, gate, post_weight, next_weight, gate_rows, scale, _ACTS[gate_act], _eps(eps, "gated_residual"), torch.is_grad_enabled())
    return y if next_weight is None else (y, u)


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
            h = self.downs[k](self.act(self.ups[k](u)))
            x, u = gated_residual(x, h, self.gates[k](u), self.posts[k], self.norms[k + 1], self.scale, "sigmoid", self.eps)
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

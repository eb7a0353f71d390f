"""8-bit quantise -> de-quantise of the grids, the evaluation-time transform of the reference
(experiment_scripts/eval.py:19-82 `quantize_keyframes`, :84-109 `quantize_sparse_grid`; the
README's 0.901 bpp operating point).  Host-side tensor glue in the reference and here (stock
torch ops, any device); arithmetic order is the reference's so results are bit-identical:

    q  = uint8( 255 * (x - min) / (max - min) + 0.5 )          (float -> uint8 truncates)
    x' = (max - min) * (float(q) / 255) + min

with min/max taken per feature and per LEVEL for the keyframes, per feature over the whole
[T,X,Y] volume for the sparse grid.

The second half of the file is 8-bit evaluation of LINEAR layers (no counterpart in the reference, whose bit budget counts the network
at 32 bits per weight, eval.py:189-190), on HIP kernels: e4m3 values with one power-of-two scale per block of 128,

    v ~ q * 2^(e - 127),  q = e4m3(v * 2^(127 - e)),  e = the smallest byte that brings the block's largest |v| to 448 or below

with a block of 128 x 128 for weights (`quantize_blocks(w, 128)`, once) and of one row x 128 columns for activations (inside the call).
`linear8(x, q, e, bias)` is the layer, `Linear8.from_linear(layer)` the module.  Inference only: there is no gradient."""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L

UNIT = 2.0 ** 8 - 1.0          # eval.py:138 unit_multiplier


def _qdq(x: torch.Tensor, lo: torch.Tensor, hi: torch.Tensor) -> torch.Tensor:
    q = (x - lo) / (hi - lo)
    q = UNIT * q
    q = torch.clamp((q + 0.5).to(torch.uint8), 0, 255)
    d = q.to(torch.float32) / UNIT
    return (hi - lo) * d + lo


def quantize_keyframes(params: torch.Tensor, config: dict) -> nn.Parameter:
    """params: flat fp32 keyframe vector -> de-quantised copy as a fresh nn.Parameter (eval.py:163-172)."""
    lv = L.make_levels(config)
    F = lv.n_features
    feats = params.detach().clone().reshape(-1, F)
    for lvl in range(lv.n_levels):
        a, b = int(lv.offset[lvl]), int(lv.offset[lvl + 1])
        blk = feats[a:b]
        for d in range(F):
            col = blk[:, d]
            feats[a:b, d] = _qdq(col, torch.min(col), torch.max(col))
    return nn.Parameter(feats.reshape(-1))


def quantize_sparse_grid(emb: torch.Tensor, config: dict | None = None) -> nn.Parameter:
    """emb [T,X,Y,F] -> de-quantised copy, per-feature global min/max (eval.py:84-109)."""
    out = emb.detach().clone()
    for d in range(out.shape[-1]):
        ch = out[..., d]
        out[..., d] = _qdq(ch, torch.min(ch), torch.max(ch))
    return nn.Parameter(out)


def quantized_bpp(model: nn.Module, n_frames: int, height: int, width: int) -> float:
    """(8 bits x every parameter + 24 extra bits x MLP parameter) / pixels   (eval.py:189-190)."""
    n_all = sum(p.numel() for p in model.parameters())
    n_mlp = sum(p.numel() for p in model.wrapper.parameters())
    return (n_all * 8 + n_mlp * 24) / (n_frames * height * width)


# --------------------------------------------------------------------------------------
# 8-bit linear layers: e4m3 with one power-of-two scale per block of 128
# --------------------------------------------------------------------------------------
BLOCK = 128


def _kblocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


def quantize_blocks(v: torch.Tensor, rows: int = 1):
    """v [R, K] (fp32 / bf16 / fp16) -> (q, e): q float8_e4m3fn [R, K rounded up to a multiple of 128] with zeros behind column K, e uint8
    [ceil(R / rows), ceil(K / 128)], v ~ q * 2^(e - 127) over blocks of `rows` (1 or 128) x 128.  Infinities and NaN become NaN and do not
    count for the block's scale; a block of zeros has e = 127."""
    if v.dim() != 2 or v.shape[1] < 1:
        raise RuntimeError(f"quantize_blocks expects a matrix with at least one column, got shape {tuple(v.shape)}")
    if rows not in (1, BLOCK):
        raise RuntimeError(f"quantize_blocks: a block has 1 or {BLOCK} rows, got {rows}")
    ty = L.stream_type(v, "quantize_blocks")
    L.binding().not_recorded("quantize_blocks")
    with L.on_device_of(v):
        v = v.detach().resolve_neg().contiguous()
        r, k = v.shape
        q = torch.empty((r, _kblocks(k) * BLOCK), device=v.device, dtype=torch.float8_e4m3fn)
        e = torch.empty(((r + rows - 1) // rows, _kblocks(k)), device=v.device, dtype=torch.uint8)
        L.check(L.load().nvp_quantize_blocks(L.ptr(v, v.dtype), ty, L.ptr(q, q.dtype), L.ptr(e, e.dtype), r, k, rows, L.stream_ptr()), "nvp_quantize_blocks")
    return q, e


def _check_blocks(q: torch.Tensor, e: torch.Tensor, k: int, rows: int, what: str) -> None:
    if q.dtype != torch.float8_e4m3fn or e.dtype != torch.uint8 or q.dim() != 2 or e.dim() != 2:
        raise RuntimeError(f"{what}: expected a float8_e4m3fn matrix and its uint8 scales, got {q.dtype} {tuple(q.shape)} and {e.dtype} {tuple(e.shape)}")
    if k < 1 or q.shape[1] != _kblocks(k) * BLOCK or tuple(e.shape) != ((q.shape[0] + rows - 1) // rows, _kblocks(k)):
        raise RuntimeError(f"{what}: {k} columns in blocks of {rows} x {BLOCK} need q [R, {_kblocks(max(k, 1)) * BLOCK}] and e [ceil(R / {rows}), {_kblocks(max(k, 1))}], "
                           f"got {tuple(q.shape)} and {tuple(e.shape)}")


def dequantize_blocks(q: torch.Tensor, e: torch.Tensor, k: int, rows: int = 1, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The matrix [R, k] that (q, e) of quantize_blocks(v, rows) stands for."""
    _check_blocks(q, e, k, rows, "dequantize_blocks")
    if rows not in (1, BLOCK):
        raise RuntimeError(f"dequantize_blocks: a block has 1 or {BLOCK} rows, got {rows}")
    L.binding().not_recorded("dequantize_blocks")
    with L.on_device_of(q, e):
        q, e = q.contiguous(), e.contiguous()                       # held until the launch: a copy that is let go is handed to the next one
        out = torch.empty((q.shape[0], k), device=q.device, dtype=dtype)
        ty = L.stream_type(out, "dequantize_blocks")
        L.check(L.load().nvp_dequantize_blocks(L.ptr(q, q.dtype), L.ptr(e, e.dtype), L.ptr(out, dtype), ty, q.shape[0], k, rows, L.stream_ptr()),
                "nvp_dequantize_blocks")
    return out


def linear8(x: torch.Tensor, q: torch.Tensor, e: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] (fp32 / bf16 / fp16) -> [..., N] of the same type: the linear layer whose weight [N, K] is (q, e) of
    quantize_blocks(weight, 128), on x quantised row by row in blocks of 128 (inside the call); products of 8-bit values, bias of x's type
    added before the one rounding.  Sums: fp32 for fp32 streams; bf16 and fp16 streams take the 8-bit matrix instruction, which adds to fp32 but drops, inside
    each group of 8 products, what lies more than 13 bits below the largest of them (2e-4 of the result's rms at the most, 1.5e-5 for normal data, where a bf16 result's own
    rounding is 1.7e-3 and an fp16 result's 2e-4).  A row with an infinity or a NaN gives a row of NaN.  Inference only."""
    return L.binding().linear8(x, q, e, bias)


class Linear8(nn.Module):
    """nn.Linear for 8-bit evaluation: holds the weight in block form (buffers `q`, `e`; 8 + 1 / 2048 bits per weight) and the bias.  The streams have the bias's
    type: a cast of the module (`half()`, `to(dtype)`) changes the bias and leaves q and e as they are."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, dtype: torch.dtype = torch.float32, device=None):
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError("Linear8 needs at least one input and one output feature")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("q", torch.zeros((out_features, _kblocks(in_features) * BLOCK), device=device, dtype=torch.float8_e4m3fn))
        self.register_buffer("e", torch.full((_kblocks(out_features), _kblocks(in_features)), 127, device=device, dtype=torch.uint8))
        self.register_buffer("bias", torch.zeros(out_features, device=device, dtype=dtype) if bias else None)

    @classmethod
    def from_linear(cls, layer: nn.Module) -> "Linear8":
        """`layer`: anything with `.weight` [N, K] and `.bias` ([N] or None) on a HIP device (nn.Linear, modulation.Siren's linear part)."""
        w, b = layer.weight.detach(), layer.bias
        m = cls(w.shape[1], w.shape[0], bias=b is not None, dtype=w.dtype, device=w.device)
        m.q, m.e = quantize_blocks(w, BLOCK)
        if b is not None:
            m.bias = b.detach().clone()
        return m

    def _apply(self, fn, recurse=True):
        """Moves go for everything; casts (`half()`, `to(dtype)`) for the bias alone: q and e are bytes, whatever type the streams have."""
        held = {n: self._buffers[n] for n in ("q", "e")}
        try:
            self._buffers.update(q=None, e=None)
            super()._apply(fn, recurse)
            moved = {n: fn(t.view(torch.uint8)) for n, t in held.items()}
            held = {n: (m if m.dtype == torch.uint8 else held[n].view(torch.uint8).to(m.device)).view(held[n].dtype) for n, m in moved.items()}
        finally:
            self._buffers.update(held)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear8(x, self.q, self.e, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

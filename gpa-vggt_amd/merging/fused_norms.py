"""The norms around a transformer block with its gate and residual, on gfx950.

`norm_gate_residual` (no counterpart in the reference) is one pass over what a
block leaves and the next one takes: the norm after the block, its gate and
residual scale, the residual, the next block's norm.  Where
`gpa::residual_layernorm` reproduces the 16-bit rounding steps of the
reference's pre-LN blocks, this one keeps fp32 between its loads and stores,
has RMS norms too, and is differentiable (`csrc/norm_gate.hip`).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native

__all__ = ["norm_gate_residual"]

_F32_MAX = torch.finfo(torch.float32).max


def _gate_rows(x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
    """The gate as [groups, C], each row of it for consecutive rows of x."""
    C = x.shape[-1]
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    lead = 0
    while lead < x.dim() - 1 and len(shape) == x.dim() and shape[lead] == x.shape[lead]:
        lead += 1
    if len(shape) != x.dim() or shape[-1] != C or any(n != 1 for n in shape[lead:-1]):
        raise ValueError(f"norm_gate_residual: gate {tuple(gate.shape)} must be [C], or x's leading "
                         f"dimensions, then ones, then C, for x {tuple(x.shape)}")
    return gate.reshape(-1, C)


def norm_gate_residual(x: torch.Tensor, y: torch.Tensor, pre_weight: torch.Tensor, *,
                       post_weight: Optional[torch.Tensor] = None,
                       post_bias: Optional[torch.Tensor] = None,
                       pre_bias: Optional[torch.Tensor] = None,
                       gate: Optional[torch.Tensor] = None, scale: float = 1.0,
                       kind: str = "rms", eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """u = N(y) * post_weight + post_bias (without post_weight: y),
    h = x + scale * gate * u, out = N(h) * pre_weight + pre_bias; returns (h, out).

    x: the residual stream, y: the block's output, both [..., C] of one type
    (GPU; fp32, bf16 or fp16; C up to 8192).  N is the RMS norm
    (kind "rms") or LayerNorm ("layer") over C.  Weights and biases are [C];
    the gate is [C], or has x's leading dimensions up to some point, ones, and C
    ([B, 1, C]: a gate for each sequence).  Parameters are of x's type, or any
    are fp32 and all are used so.  Inside everything is fp32; h and out are
    rounded once each, out from the unrounded h.  Differentiable in all tensors.
    """
    what = "norm_gate_residual"
    if kind not in ("rms", "layer"):
        raise ValueError(f"{what}: kind {kind!r} is not 'rms' or 'layer'")
    if not (0 <= eps <= _F32_MAX and abs(scale) <= _F32_MAX):
        raise ValueError(f"{what}: eps must be finite and >= 0, scale finite, in fp32, got {eps} and {scale}")
    if not 1 <= x.dim() or x.shape != y.shape:
        raise ValueError(f"{what}: x {tuple(x.shape)} and y {tuple(y.shape)} differ")
    if x.shape[-1] > 8192 or x.shape[-1] < 1:
        raise NotImplementedError(f"{what}: {x.shape[-1]} features (1 to 8192)")
    if gate is not None:
        gate = _gate_rows(x, gate)
    par = (post_weight, post_bias, gate, pre_weight, pre_bias)
    if any(t is not None and t.dtype != x.dtype for t in par):
        par = tuple(None if t is None else t.float() for t in par)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, *par))
    h, out, _ = _native.norm_gate(x, y, *par, float(scale), kind == "layer", float(eps), grad)
    return h, out

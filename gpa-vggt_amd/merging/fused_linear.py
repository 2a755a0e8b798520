"""A block's projections with what follows them, on gfx950.

`linear_gate_residual` (no counterpart in the reference) is a product with its
bias, activation, per-feature gate and residual in one pass, differentiable
(`csrc/linear_gate.hip`): the projections and the two products of a block's MLP,
beside the norms of `merging.fused_norms` and the attention of
`merging.fused_attention`.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .fused_attention import _half_operands

__all__ = ["linear_gate_residual"]

_ACTS = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "relu": 4}


def linear_gate_residual(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                         activation: Optional[str] = None, gate: Optional[torch.Tensor] = None,
                         residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + gate * activation(x weight^T + bias).

    x [..., K], weight [N, K] (GPU, bf16 or fp16; an fp32 x is cast to the autocast dtype or
    bf16, and residual with it; weight is used in x's type; any strides), bias and gate [N],
    residual [..., N] of x's type (a wider one would lose what it has more: it is refused, and
    added outside).
    activation: None, "gelu" (the normal distribution's), "gelu_tanh", "silu" or "relu".  bias
    and gate are of x's type, or any is fp32 and both are used so.  From the products to
    the result everything is fp32; it is rounded once.  Returns [..., N]; differentiable in all
    tensors (dz, the gradient before the activation, is rounded to x's type for its two products).

    Where K is no multiple of 8, or rows are not 16-byte aligned, x and weight are first
    copied into padded rows.
    """
    what = "linear_gate_residual"
    if activation not in _ACTS:
        raise ValueError(f"{what}: activation {activation!r} is not one of {sorted(a for a in _ACTS if a)} or None")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    N, lead = weight.shape[0], x.shape[:-1]
    if residual is not None and residual.shape != (*lead, N):
        raise ValueError(f"{what}: residual {tuple(residual.shape)} must be {(*lead, N)}")
    if residual is not None and residual.dtype != x.dtype and x.dtype in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: residual is {residual.dtype} beside x in {x.dtype}; cast one of them")
    x, weight = _half_operands(x, (weight,))
    if residual is not None and residual.dtype != x.dtype:
        residual = residual.to(x.dtype)
    if (bias is not None and bias.dtype != x.dtype) or (gate is not None and gate.dtype != x.dtype):
        bias, gate = (None if t is None else t.float() for t in (bias, gate))
    act = _ACTS[activation]
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, gate, residual))
    flat = lambda t, n: t if t is None or t.dim() == 2 else t.reshape(lead.numel(), n)  # noqa: E731
    y, _ = _native.linear_gate(flat(x, x.shape[-1]), weight, bias, gate, flat(residual, N), act,
                               grad and (act > 0 or gate is not None))
    return y if x.dim() == 2 else y.view(*lead, N)

"""Flash attention with a per-key additive bias, on gfx950.

Drop-in for the reference's `merging/fused_attention.py`: same function name,
arguments, dtype contract and return types (`attention_keybias`, reference
:130-180) and the same `LOG2E` constant (:40).  The kernel is the
hand-written HIP kernel `attn_keybias_kernel` in `csrc/attn_keybias.hip`,
reached through the `gpa::attn_keybias` custom op.

Math matches SDPA(q, k, v, attn_mask=bias): scores = q@k^T * scale + bias,
softmax over keys in fp32, P rounded to the operand format (bf16 or fp16)
for the P@V product, fp32 accumulation.  With return_lse the log2 softmax
denominators come back as well, so callers can split the key set and
recombine exactly (reference :123-127); `combine_by_lse` is that recombination for the
frame-special split path of vggt/layers/attention.py:148-176.

`attention_masked` and `attention_shared_prefix` (no counterpart in the
reference) are the attention of language-model blocks: packed documents,
causal and prefix masks, capped and distance-biased scores, shared key heads,
gradients, and a prefix that a whole batch shares (`csrc/attn_masked.hip`).
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native

__all__ = ["attention_keybias", "attention_join", "attention_masked", "attention_rows",
           "attention_shared_prefix", "combine_by_lse", "LOG2E"]

LOG2E = 1.4426950408889634
_F32_MIN, _F32_MAX = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def _autocast_dtype() -> torch.dtype:
    if torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda")
    return torch.bfloat16


def _operands(q, k, v, bias):
    if q.dtype == torch.float32:
        dt = _autocast_dtype()
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
        bias = None if bias is None else bias.to(dt)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(
            f"attention_keybias: {q.dtype} is not supported; the gfx950 kernels run bf16 and fp16")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention_keybias expects [B, H, T, D] q/k/v")
    return q, k.to(q.dtype), v.to(q.dtype), bias


def attention_keybias(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      bias: torch.Tensor, sm_scale: float, return_lse: bool = False):
    """SDPA(q, k, v, attn_mask=bias) where bias is per-key: [B, H, 1, N].

    q [B, H, M, D], k/v [B, H, N, D] (GPU, bf16 or fp16; fp32 inputs are cast
    to the autocast dtype or bf16 first, as at merging/fused_attention.py:
    139-144).  Returns [B, H, M, D] in q's dtype; with return_lse also
    [B, H, M] fp32 log2 softmax denominators.  `bias` may be None (plain
    attention).
    """
    q, k, v, bias = _operands(q, k, v, bias)
    o, lse = _native.attn_keybias(q, k, v, bias, float(sm_scale), bool(return_lse))
    return (o, lse) if return_lse else o


def attention_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   bias: Optional[torch.Tensor], sm_scale: float) -> torch.Tensor:
    """`attention_keybias` as the [B, M, H*D] rows the output projection takes."""
    return _native.attn_keybias_rows(*_operands(q, k, v, bias), float(sm_scale))


def attention_join(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   bias: Optional[torch.Tensor], sm_scale: float, out_a: torch.Tensor,
                   lse_a: torch.Tensor, frames: int) -> torch.Tensor:
    """`attention_keybias` of all queries over the shared keys and
    `combine_by_lse` with the own-frame half (out_a, lse_a), in one pass at head
    dim 64, where the shared half then stays in fp32."""
    q, k, v, bias = _operands(q, k, v, bias)
    if q.shape[-1] == 64 and out_a.dtype == q.dtype:
        return _native.attn_keybias_join(q, k, v, bias, float(sm_scale), out_a, lse_a, int(frames))
    out_b, lse_b = _native.attn_keybias(q, k, v, bias, float(sm_scale), True)
    return combine_by_lse(out_a, lse_a, out_b, lse_b, frames)


def combine_by_lse(out_a: torch.Tensor, lse_a: torch.Tensor, out_b: torch.Tensor,
                   lse_b: torch.Tensor, frames: int) -> torch.Tensor:
    """Merge the two halves of the frame-special split attention.

    out_a [B*S, H, P, D], lse_a [B*S, H, P]: attention of every frame's P
    queries over the frame's own keys (frame-major, as the own-frame call of
    vggt/layers/attention.py:157 returns it); out_b [B, H, S*P, D], lse_b
    [B, H, S*P]: attention of all queries over the shared keys (:162).  The
    log2 LSEs weight the two (:166-176); returns [B, S*P, H*D] in the
    outputs' dtype (bf16 or fp16), the layout the output projection takes.
    The weights and the sum are fp32 (the reference rounds the weights to the
    activation dtype first).
    """
    return _native.lse_combine(out_a, lse_a, out_b, lse_b, int(frames))


def _score_args(what, sm_scale, cap, slopes):
    sm_scale = float(sm_scale)
    if not _F32_MIN <= sm_scale <= _F32_MAX:
        raise ValueError(f"{what}: sm_scale must be finite and positive in fp32, got {sm_scale}")
    if cap is not None and not _F32_MIN <= cap <= _F32_MAX:
        raise ValueError(f"{what}: cap must be finite and positive in fp32, or None, got {cap}")
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: the slopes are constants (they have no gradient)")
    return sm_scale, 0.0 if cap is None else float(cap)


def _half_operands(q, others):
    if q.dtype == torch.float32:
        q = q.to(_autocast_dtype())
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{q.dtype} is not supported; the gfx950 kernels run bf16 and fp16")
    return (q, *(t.to(q.dtype) for t in others))


def attention_masked(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sm_scale: float, *,
                     cap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
                     causal: bool = False, prefix: Union[None, int, torch.Tensor] = None,
                     offsets: Optional[torch.Tensor] = None,
                     k_offsets: Optional[torch.Tensor] = None, return_lse: bool = False):
    """softmax(s) v over the keys that each query sees, differentiable in q, k and v.

    q [B, H, M, D], k and v [B, Hk, N, D] (GPU, bf16 or fp16, fp32 inputs cast
    as in `attention_keybias`; D 64 or 128; any strides): query head h reads
    key head h // (H // Hk).

    x = sm_scale q.k;  s = cap tanh(x / cap) (cap None: x), less
    slopes[h] * |p_q - p_k| (slopes fp32 [H] or [B, H], of either sign, constants).

    Documents: run d holds the queries offsets[d] .. offsets[d + 1] - 1 and the
    keys of k_offsets likewise (int32 [docs + 1], or [B, docs + 1] where they
    differ by batch element; k_offsets None: the same as the queries', which
    then need N = M).  Without offsets there is one document of all queries
    and the keys of k_offsets (a padded batch: [[0, length], ...]), or of all
    keys.  Positions count from a document's first key, and its last query
    stands at its last key, as new tokens at the end of a cache do.  `causal`:
    a query sees the keys up to its position and the first `prefix` ones of
    its document (a number, or int32 [docs] or [B, docs]).  A query that
    sees nothing, and a token of no document, gets zeros (LSE -inf) and
    no gradient.  Offsets are read on the GPU: they must not decrease, and
    what lies outside the tensors is cut to them.

    Returns [B, H, M, D] in q's dtype (of an fp32 q: what it was cast to) and order
    of dimensions; with return_lse also the log2 softmax denominators [B, H, M] fp32.
    """
    what = "attention_masked"
    sm_scale, cap = _score_args(what, sm_scale, cap, slopes)
    q, k, v = _half_operands(q, (k, v))
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{what} expects [B, H, T, D] q/k/v")
    if offsets is not None and k_offsets is None:
        if k.shape[2] != q.shape[2]:
            raise ValueError(f"{what}: {q.shape[2]} queries and {k.shape[2]} keys need k_offsets too")
        k_offsets = offsets
    for name, t in (("offsets", offsets), ("k_offsets", k_offsets)):
        if t is not None and (t.dim() not in (1, 2) or t.shape[-1] < 2):
            raise ValueError(f"{what}: {name} must hold docs + 1 values, got {tuple(t.shape)}")
    if offsets is None and k_offsets is not None and k_offsets.shape[-1] != 2:
        raise ValueError(f"{what}: {k_offsets.shape[-1] - 1} documents of keys need the queries' offsets")
    prefix_len = 0
    if prefix is not None:
        if not causal:
            raise ValueError(f"{what}: a prefix goes with the causal mask")
        if not isinstance(prefix, torch.Tensor):
            prefix, prefix_len = None, int(prefix)
            if prefix_len < 0:
                raise ValueError(f"{what}: prefix {prefix_len} is negative")
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    o, lse, _ = _native.attn_masked(q, k, v, sm_scale, cap, slopes, bool(causal), prefix, prefix_len,
                                 offsets, k_offsets, bool(return_lse) or grad, bool(return_lse), grad)
    return (o, lse) if return_lse else o


def attention_shared_prefix(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor,
                            k: torch.Tensor, v: torch.Tensor, sm_scale: float, *,
                            lengths: Optional[torch.Tensor] = None, cap: Optional[float] = None,
                            slopes: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal attention of a batch over a prefix that all its sequences share
    and the keys of their own, the prefix read once for all of them.

    prefix_k, prefix_v [Hk, P, D]; k, v [B, Hk, N, D], of which lengths[b]
    (int32 [B]; None: N) belong to sequence b, the new tokens among them;
    q [B, H, M, D]: the last M tokens of each.  Query i sees the prefix and
    the own keys up to its own, lengths[b] - M + i.  Scores, dtypes and results
    as in `attention_masked`; positions count from the prefix's first key.
    Forward only.
    """
    what = "attention_shared_prefix"
    sm_scale, cap = _score_args(what, sm_scale, cap, slopes)
    q, prefix_k, prefix_v, k, v = _half_operands(q, (prefix_k, prefix_v, k, v))
    o, lse = _native.attn_shared_prefix(q, prefix_k, prefix_v, k, v, lengths, sm_scale, cap, slopes,
                                        bool(return_lse))
    return (o, lse) if return_lse else o

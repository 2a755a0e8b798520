"""Norms of query and key heads and their rotation by positions, on gfx950.

`qk_norm_rotate` and `rotate_heads` (no counterpart in the reference) are what
queries and keys go through between a block's projection and its attention
(`csrc/head_rotary.hip`).  Where `gpa::qk_norm_rope` reproduces the
aggregator's LayerNorm and two-axis rotation of 64-feature heads from host
tables, these take any even head dim, RMS norms too, shared key heads,
positions of up to eight axes (time, height and width of video tokens) as far
as they reach, and are differentiable.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _native

__all__ = ["RotaryAxes", "qk_norm_rotate", "rotary_axes", "rotate_heads"]

_F32_MAX = torch.finfo(torch.float32).max
_PAIRINGS = {"half": 0, "interleaved": 1, "blocks": 2}
_NORMS = {"rms": 1, "layer": 2}


class RotaryAxes(NamedTuple):
    """Which features turn, by which axis of the positions and how fast.

    freqs: fp64 [pairs], radians a unit of position; axes: int32 [pairs], the
    column of the positions that a pair turns by (both on the GPU); sections:
    the pairs of each axis (they add to `pairs`).  pairing: feature j turns
    with pairs + j ("half"), 2 j with 2 j + 1 ("interleaved"), or the features
    of each axis's own block, of twice its section, in halves ("blocks": pairs
    then are in the order of the sections).  Features past 2 * pairs stay.
    """
    freqs: torch.Tensor
    axes: torch.Tensor
    pairing: str
    sections: Tuple[int, ...]


def rotary_axes(sections: Sequence[int], *, base: float = 10000.0, ladder: str = "shared",
                pairing: str = "half", order: str = "sections", device="cuda") -> RotaryAxes:
    """The usual geometric frequencies for len(sections) axes.

    ladder "shared": one ladder base^(-j / pairs) over all pairs, of which each
    axis has some; "own": base^(-i / section) for each axis.  order "sections":
    an axis has consecutive pairs; "dealt": the axes take pairs in turn until
    their sections are used up (with the shared ladder each then has fast and
    slow ones).
    """
    sections = tuple(int(s) for s in sections)
    if not 1 <= len(sections) <= _native.MAX_AXES or any(s < 0 for s in sections):
        raise ValueError(f"rotary_axes: 1 to {_native.MAX_AXES} sections of 0 or more pairs, got {sections}")
    if ladder not in ("shared", "own") or pairing not in _PAIRINGS or order not in ("sections", "dealt"):
        raise ValueError(f"rotary_axes: unknown ladder {ladder!r}, pairing {pairing!r} or order {order!r}")
    if pairing == "blocks" and order != "sections":
        raise ValueError("rotary_axes: blocks hold the pairs of one axis each (order 'sections')")
    if not 0 < base <= _F32_MAX:
        raise ValueError(f"rotary_axes: base must be finite and positive, got {base}")
    pairs = sum(sections)
    if order == "sections":
        axes = [a for a, s in enumerate(sections) for _ in range(s)]
    else:
        axes = [a for i in range(max(sections)) for a, s in enumerate(sections) if i < s]
    seen, freqs = [0] * len(sections), []
    for j, a in enumerate(axes):
        freqs.append(float(base) ** (-seen[a] / sections[a] if ladder == "own" else -j / pairs))
        seen[a] += 1
    return RotaryAxes(torch.tensor(freqs, dtype=torch.float64, device=device),
                      torch.tensor(axes, dtype=torch.int32, device=device), pairing, sections)


def _parts(what, rotary, positions):
    if (rotary is None) != (positions is None):
        raise ValueError(f"{what}: positions go with the rotation")
    if rotary is None:
        return None, None, 0, []
    if rotary.pairing not in _PAIRINGS:
        raise ValueError(f"{what}: pairing {rotary.pairing!r} is not one of {sorted(_PAIRINGS)}")
    if positions.requires_grad or rotary.freqs.requires_grad:
        raise ValueError(f"{what}: positions and frequencies are constants (they have no gradient)")
    return rotary.freqs, rotary.axes, _PAIRINGS[rotary.pairing], list(rotary.sections)


def _heads_checked(what, q, k=None):
    for t in (q, k):
        if t is not None and t.dim() != 4:
            raise ValueError(f"{what} expects [B, H, N, D] tensors, got {tuple(t.shape)}")
        if t is not None and (t.shape[3] % 2 or not 2 <= t.shape[3] <= 256):
            raise NotImplementedError(f"{what}: head dim {t.shape[3]} (even, 2 to 256)")


def rotate_heads(x: torch.Tensor, positions: torch.Tensor, rotary: RotaryAxes) -> torch.Tensor:
    """x [B, H, N, D] (GPU; fp32, bf16 or fp16; any strides; D even, up to 256)
    with its pairs of features (a, b) turned by t = positions[n, axis] * freq:
    (a cos t - b sin t, b cos t + a sin t).

    positions [N, axes] or [B, N, axes], int32, int64 or fp32, constants, of any
    size: angles are formed in 64 bits.  Returns x's type and order of
    dimensions, rounded once; differentiable in x.
    """
    what = "rotate_heads"
    _heads_checked(what, x)
    return _native.head_rotary(x, None, positions, *_parts(what, rotary, positions), None, None, None,
                               None, 0, 0.0)[0]


def qk_norm_rotate(q: torch.Tensor, k: torch.Tensor, positions: Optional[torch.Tensor],
                   rotary: Optional[RotaryAxes], *, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, q_bias: Optional[torch.Tensor] = None,
                   k_bias: Optional[torch.Tensor] = None, kind: str = "rms",
                   eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """Every head of q [B, H, N, D] and k [B, Hk, N, D] normed over its D
    features (kind "rms" or "layer"), times weight plus bias ([D], shared by
    the tensor's heads; None: 1 and 0), then turned as in `rotate_heads` (rotary and
    positions None: not turned), in one pass.

    Parameters are of q's type, or any are fp32 and all are used so.  Inside
    everything is fp32, and each output is rounded once.  Differentiable in q, k and the
    parameters; returns tensors in q's and k's order of dimensions, as the
    framework's attention takes them.
    """
    what = "qk_norm_rotate"
    if kind not in _NORMS:
        raise ValueError(f"{what}: kind {kind!r} is not 'rms' or 'layer'")
    if not 0 <= eps <= _F32_MAX:
        raise ValueError(f"{what}: eps must be finite and >= 0 in fp32, got {eps}")
    _heads_checked(what, q, k)
    freqs, axes, pairing, sections = _parts(what, rotary, positions)
    par = (q_weight, k_weight, q_bias, k_bias)
    if any(t is not None and t.dtype != q.dtype for t in par):
        par = tuple(None if t is None else t.float() for t in par)
    return _native.head_rotary(q, k, positions, freqs, axes, pairing, sections, *par, _NORMS[kind], float(eps))

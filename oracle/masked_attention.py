"""64-bit masked attention with its gradients and error bounds (test
infrastructure only).

Plain loops over batch elements, documents and heads, with an explicit mask:
the definition that `attention_masked` documents, written apart from the
kernels' ranges.  `bounds` says how far 16-bit operands and outputs may
take a result: P, dS and the outputs are each rounded once (`u`, half a step
of the format), scores and sums are fp32.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

LOG2E = 1.4426950408889634


class Result(NamedTuple):
    o: torch.Tensor
    lse: torch.Tensor
    dq: Optional[torch.Tensor]
    dk: Optional[torch.Tensor]
    dv: Optional[torch.Tensor]
    o_bound: torch.Tensor
    dq_bound: Optional[torch.Tensor]
    dk_bound: Optional[torch.Tensor]
    dv_bound: Optional[torch.Tensor]
    lse_bound: float


def _per_batch(x, b):
    return x[b] if isinstance(x[0], (list, tuple)) else x


def masked_attention(q, k, v, sm_scale, *, cap=None, slopes=None, causal=False, prefix=0,
                     offsets=None, k_offsets=None, d_o=None, d_lse=None, u=2.0 ** -8) -> Result:
    """q [B,H,M,D], k/v [B,Hk,N,D] on the CPU; offsets are lists (or one list a
    batch element), prefix a number or a list by document."""
    B, H, M, D = q.shape
    Hk, N = k.shape[1], k.shape[2]
    q, k, v = q.double(), k.double(), v.double()
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    o, lse = z(B, H, M, D), torch.full((B, H, M), -math.inf, dtype=torch.float64)
    ob, lse_b = z(B, H, M, D), 0.0
    back = d_o is not None or d_lse is not None
    dq, dk, dv, dqb, dkb, dvb = (z(*t.shape) if back else None for t in (q, k, v, q, k, v))
    if back:
        d_o = torch.zeros_like(q) if d_o is None else d_o.double()
        d_lse = z(B, H, M) if d_lse is None else d_lse.double()
    if k_offsets is None:
        k_offsets = offsets
    f = 2.0 ** -24
    for b in range(B):
        qo = [0, M] if offsets is None else _per_batch(offsets, b)
        ko = [0, N] if k_offsets is None else _per_batch(k_offsets, b)
        for d in range(len(qo) - 1):
            rows, keys = slice(qo[d], qo[d + 1]), slice(ko[d], ko[d + 1])
            m, n = qo[d + 1] - qo[d], ko[d + 1] - ko[d]
            if m <= 0 or n <= 0:
                continue
            at = torch.arange(n - m, n, dtype=torch.float64)[:, None]
            j = torch.arange(n, dtype=torch.float64)[None]
            pre = prefix[d] if isinstance(prefix, (list, tuple)) else prefix
            seen = (j <= at) | (j < pre) if causal else torch.ones(m, n, dtype=torch.bool)
            for h in range(H):
                g = h // (H // Hk)
                qh, kh, vh = q[b, h, rows], k[b, g, keys], v[b, g, keys]
                x = qh @ kh.T * sm_scale
                size = (qh.abs() @ kh.abs().T).max().item() * sm_scale
                t = torch.tanh(x / cap) if cap else None
                s = cap * t if cap else x
                err = (D + 8) * f * size + (16 * f * cap if cap else 0.0)
                if slopes is not None:
                    sl = float(slopes[b][h] if slopes.dim() == 2 else slopes[h])
                    s = s - sl * (at - j).abs()
                    err += 4 * f * abs(sl) * max(n, m)
                s = s.masked_fill(~seen, -math.inf)
                ls = torch.logsumexp(s, -1)
                p = torch.exp(s - ls.clamp_min(-1e300)[:, None])
                p = torch.where(seen, p, torch.zeros_like(p))
                err = 4 * err + (n + 64) * f           # of a weight, relative
                lse_b = max(lse_b, err * LOG2E + 2 * f * float(ls[ls > -math.inf].abs().max() if (ls > -math.inf).any() else 0) * LOG2E)
                oh = p @ vh
                o[b, h, rows], lse[b, h, rows] = oh, ls * LOG2E
                ob[b, h, rows] = u * oh.abs() + (u + 2 * err) * (p @ vh.abs()) + 1e-30
                if not back:
                    continue
                go, gl = d_o[b, h, rows], d_lse[b, h, rows]
                dp = go @ vh.T
                delta = (go * oh).sum(-1, keepdim=True) - LOG2E * gl[:, None]
                der = sm_scale * (1 - t * t if cap else torch.ones_like(x))
                ds = p * (dp - delta) * der
                # delta is formed from the rounded output, dP and delta in fp32
                off = (go.abs() * ob[b, h, rows]).sum(-1, keepdim=True)
                mag = go.abs() @ vh.abs().T + (go.abs() * oh.abs()).sum(-1, keepdim=True) + LOG2E * gl.abs()[:, None]
                dsb = (u + 4 * err) * ds.abs() + p * (off + (D + 8) * f * mag) * der.abs() + 16 * f * p * mag * sm_scale
                dq[b, h, rows] += ds @ kh
                dk[b, g, keys] += ds.T @ qh
                dv[b, g, keys] += p.T @ go
                dqb[b, h, rows] += dsb @ kh.abs()
                dkb[b, g, keys] += dsb.T @ qh.abs()
                dvb[b, g, keys] += (u + 2 * err) * (p.T @ go.abs())
    if back:
        dqb, dkb, dvb = (bound + u * g.abs() + 1e-30 for bound, g in ((dqb, dq), (dkb, dk), (dvb, dv)))
    return Result(o, lse, dq, dk, dv, ob, dqb, dkb, dvb, lse_b + 1e-6)

"""Gradients of `linear_gate_residual` where an activation's slope is small and steep beside its size:
the kept sums are near enough for it.

f = 2^-24, u half a step of the type.  A sum of K products and a bias is off by ze = (K + 16) f of their
sizes, which moves the slope by its derivative there (1.1 times for what that changes on the way);
`_act` has the slope's own error.  dz is rounded once for dw's product, dbias is fp32's sum of the unrounded."""
import pytest
import torch

from merging.fused_linear import linear_gate_residual
from test_gpu_linear_gate import _act

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
f = 2.0 ** -24


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,N", [(400, 64), (9, 64), (400, 61)])
@pytest.mark.parametrize("act,at", [("silu", (-3.3, -8.3, -10.7, -14.2, 9.1)), ("gelu", (-0.76, -2.3, -3.1, 2.9)),
                                    ("gelu_tanh", (-0.76, -2.3, -3.1, 2.9))])
def test_slopes_of_sums_that_a_bias_sets(dev, dt, M, N, act, at):
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    K, u, tiny = 16, torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == HF else 0.0
    x, w, dy = (r(M, K) / 64).to(dt), (r(N, K) / 64).to(dt), (r(M, N).abs() + 0.5).to(dt)
    b = torch.tensor(at, device=dev).repeat(-(-N // len(at)))[:N] + 0.01 * r(N)
    leaves = [w.requires_grad_(), b.requires_grad_()]
    dw, db = torch.autograd.grad(linear_gate_residual(x, *leaves, activation=act), leaves, dy)
    x, w, b, dy = (t.detach().double() for t in (x, w, b, dy))
    z, ze = (x @ w.t() + b).requires_grad_(), (K + 16) * f * (x.abs() @ w.abs().t() + b.abs())
    _, slope, _, se = _act(z, act)
    second, = torch.autograd.grad(slope.sum(), z)
    dz, off = (dy * slope).detach(), dy * (se.detach() + 1.1 * second.abs() * ze) + 4 * f * (dy * slope.detach()).abs()
    want = dz.sum(0)
    bound = off.sum(0) + (M + 64) * f * dz.abs().sum(0) + f * want.abs()
    bad = (db.double() - want).abs() / bound
    assert bad.max() <= 1, f"dbias: worst {float(bad.max()):.3g} bounds"
    want = dz.t() @ x
    bound = u * want.abs() + (off + u * (dz.abs() + off) + tiny).t() @ x.abs() + (M + 16) * f * (dz.abs().t() @ x.abs()) + tiny
    bad = (dw.double() - want).abs() / bound
    assert bad.max() <= 1, f"dw: worst {float(bad.max()):.3g} bounds"

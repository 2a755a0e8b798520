"""fp16 gradients of `linear_gate_residual` under gates of very unequal size.

As in the projections' other tests, u = 2^-11 is half a step of fp16 relative to a value, tiny = 2^-25
half its smallest step, and f = 2^-24.  dw's row of a gate g comes from dy act'(z), rounded once (u of
it, tiny at least) and g times the sum; dx's row from dy g act'(z), rounded once after a power of two
that brings the row's largest |dy g| to 2^13 or more (u, and tiny / 2^13 of that largest at least)."""
import pytest
import torch

from merging.fused_linear import linear_gate_residual
from test_gpu_linear_gate import _act

pytestmark = pytest.mark.gpu
F, HF = torch.float32, torch.float16
f, u, tiny = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25


def _check(dev, M, N, K, gate, pdt, act, size, only_small=False, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    gate = torch.tensor(gate, device=dev).repeat(-(-N // len(gate)))[:N].to(pdt)
    x, w, dy = (1.1 * r(M, K)).to(HF), (r(N, K) * K ** -0.5).to(HF), (size * r(M, N)).to(HF)
    if only_small:                                           # nothing comes in but through the smallest gates
        dy = torch.where(gate == gate.min(), dy, 0)
    leaves = [t.requires_grad_() for t in (x, w)]
    dx, dw = torch.autograd.grad(linear_gate_residual(x, w, gate=gate, activation=act), leaves, dy)
    x, w, dy, gate = (t.detach().double() for t in (x, w, dy, gate))
    z, ze = x @ w.t(), (K + 16) * f * (x.abs() @ w.abs().t())
    _, slope, _, se = _act(z, act)
    bare = dy * slope
    off = dy.abs() * (se + 1.2 * ze) + 4 * f * bare.abs() if act else bare * 0
    dz, dz_off = bare * gate, off * gate.abs()
    want = bare.t() @ x * gate[:, None]
    rounded = off + u * (bare.abs() + off) + tiny
    bound = u * want.abs() + (rounded.t() @ x.abs() + (M + 16) * f * (bare.abs().t() @ x.abs())) * gate.abs()[:, None] + tiny
    bad = (dw.double() - want).abs() / bound
    assert bad.max() <= 1, f"dw: worst {float(bad.max()):.3g} bounds, gate {float(gate[bad.amax(1).argmax()]):.3g}"
    least = tiny * 2.0 ** -13 * (dy * gate).abs().amax(1, keepdim=True)
    want = dz @ w
    rounded = dz_off + u * (dz.abs() + dz_off) + least
    bound = u * want.abs() + rounded @ w.abs() + (N + 16) * f * (dz.abs() @ w.abs()) + tiny
    bad = (dx.double() - want).abs() / bound
    assert bad.max() <= 1, f"dx: worst {float(bad.max()):.3g} bounds"


@pytest.mark.parametrize("act", [None, "silu", "relu"])
@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("gate,pdt", [((300.0, 0.3), HF), ((300.0, 30.0, 3.0, 0.3, 0.03, 0.003), HF), ((1e4, 1.0, 1e-4), F),
                                      ((1.0, 1e-5), F)])
def test_gates_over_decades(dev, act, size, gate, pdt):
    _check(dev, 2048, 64, 80, gate, pdt, act, size)
    _check(dev, 300, 63, 77, gate, pdt, act, size)


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("N", [72, 71])
def test_rows_that_the_large_gates_do_not_reach(dev, act, N):
    _check(dev, 200, N, 64, (1e4, 1e-3), F, act, 1e-2, only_small=True)


def test_rows_of_unequal_size(dev):
    """A row's scale is its own: rows 2^20 apart, one of zeros and one of fp16's largest among them."""
    g = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    w, gate = (r(40, 24) / 8).to(HF), torch.tensor([1e-3, 0.2], device=dev).repeat(20)
    dy = (r(70, 40).clamp(-3, 3) * 2.0 ** torch.linspace(-12, 8, 70, device=dev)[:, None]).to(HF)
    dy[3], dy[9] = 0, 65504
    x = r(70, 24).to(HF).requires_grad_()
    dx, = torch.autograd.grad(linear_gate_residual(x, w, gate=gate), x, dy)
    dz = dy.double() * gate.double()
    want, least = dz @ w.double(), tiny * 2.0 ** -13 * dz.abs().amax(1, keepdim=True)
    bound = u * want.abs() + (u * dz.abs() + least) @ w.double().abs() + 56 * f * (dz.abs() @ w.double().abs()) + tiny
    assert ((dx.double() - want).abs() <= bound).all() and not dx[3].any()


@pytest.mark.parametrize("want", [(0,), (1,), (0, 1)])
def test_each_gradient_alone(dev, want):
    """dx and dw do not depend on what else is wanted."""
    g = torch.Generator(device=dev).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(HF)  # noqa: E731
    ts, dy = [r(130, 64), r(72, 64), r(72), r(72) * 100], r(130, 72) / 64

    def grads(which):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate(ts)]
        y = linear_gate_residual(*leaves[:3], gate=leaves[3], activation="gelu_tanh")
        return dict(zip(which, torch.autograd.grad(y, [leaves[i] for i in which], dy)))
    every, some = grads((0, 1, 2, 3)), grads(want)
    assert all(torch.equal(some[i], every[i]) for i in want)

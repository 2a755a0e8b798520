"""Gradients of `linear_gate_residual` whose operands' rows lie over each other: the product over rows
takes no more of them than there are.

x, w and dy hold whole numbers up to 4, so that every sum here is below 2^24 and exact in fp32: the
gradients are the definition's, rounded once."""
import ctypes

import pytest
import torch

from merging import _native
from merging.fused_linear import linear_gate_residual

FAKE = 4096
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("kw,g,copied", [
    (dict(x_s=0), {}, 300 * 128 * 2), (dict(x_s=120), {}, 300 * 128 * 2), (dict(w_s=0), {}, 64 * 128 * 2),
    (dict(w_s=8), {}, 64 * 128 * 2), ({}, dict(dy_s=0), 300 * 64 * 2), ({}, dict(dy_s=56), 300 * 64 * 2),
    (dict(M=1, x_s=0), dict(dy_s=0), 0), (dict(N=1 << 3, w_s=128), dict(dy_s=8), 0)])
def test_copies_of_rows_that_overlap(kw, g, copied):
    """They are in the workspace, whose size tells; a single row does not overlap, nor do rows that touch."""
    def need(kw, g):
        a, grads = _native._LinearArgs(), _native._LinearGrads()
        for name, x in {**dict(x=FAKE, w=FAKE, bias=FAKE, M=300, N=64, K=128, x_s=128, w_s=128), **kw}.items():
            setattr(a, name, x)
        for name, x in {**dict(dy=FAKE, dx=FAKE, dw=FAKE, dy_s=a.N, dx_s=128, dw_s=128), **g}.items():
            setattr(grads, name, x)
        return _native.lib().gpa_linear_gate_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(grads))
    apart = {k: v for k, v in kw.items() if k not in ("x_s", "w_s")}
    assert need(kw, g) == need(apart, {}) + copied


def _whole(g, dev, dt, *shape):
    return torch.randint(-4, 5, shape, generator=g, device=dev).to(dt)


def _rows(g, dev, dt, R, C, how):
    """[R, C]: rows of their own, one row R times, or windows eight values apart."""
    if how == "own":
        return _whole(g, dev, dt, R, C)
    if how == "one":
        return _whole(g, dev, dt, 1, C).expand(R, C)
    return _whole(g, dev, dt, 8 * (R - 1) + C).as_strided((R, C), (8, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M", [2, 8, 40, 70, 300])
@pytest.mark.parametrize("x_rows", ["own", "one", "windows"])
@pytest.mark.parametrize("dy_rows", ["own", "one", "windows"])
def test_gradients_of_rows_that_overlap(dev, dt, M, x_rows, dy_rows):
    g = torch.Generator(device=dev).manual_seed(M)
    x, w = _rows(g, dev, dt, M, 64, x_rows), _rows(g, dev, dt, 40, 64, "windows")
    dy = _rows(g, dev, dt, M, 40, dy_rows)
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    y = linear_gate_residual(*leaves)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, (x.double() @ w.double().t()).to(dt))
    assert torch.equal(dx, (dy.double() @ w.double()).to(dt))
    assert torch.equal(dw, (dy.double().t() @ x.double()).to(dt))


@pytest.mark.gpu
def test_infinities_of_rows_that_overlap(dev):
    """An infinity of a repeated row meets the rows' own gradients alone, none of them zero."""
    g = torch.Generator(device=dev).manual_seed(1)
    x = _whole(g, dev, BF, 40, 64)
    w = _whole(g, dev, BF, 1, 64)
    w[0, 3] = torch.inf
    dy = torch.ones(40, 40, device=dev, dtype=BF)
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(linear_gate_residual(leaf, w.expand(40, 64)), leaf, dy)
    want = (dy.double() @ w.expand(40, 64).double()).to(BF)
    assert (want[:, 3] == torch.inf).all() and torch.equal(dx, want)

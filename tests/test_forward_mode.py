"""No op has a forward-mode derivative: a tangent is refused, by the callables and by the registered
ops, eagerly and under transforms.  (Below autograd it would be dropped, and a jvp be zero.)"""
import functools
from typing import Tuple

import pytest
import torch
from torch.autograd import forward_ad

from merging import _native
from merging.fused_attention import attention_masked, attention_tree, draft_tree
from merging.fused_linear import linear_gate_residual
from merging.fused_norms import norm_gate_residual
from merging.fused_rotary import qk_norm_rotate, rotary_axes, rotate_heads

BF = torch.bfloat16
ANYWHERE = pytest.mark.parametrize("where", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def _times(x, s):
    return x * s, x.sum()


def tangent_probe(x: torch.Tensor, s: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return _times(x, s)


def tangent_probe_far(x: torch.Tensor, s: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return _times(x, s)


@functools.partial(_native._op, direct=True)
def tangent_probe_forward(x: torch.Tensor, s: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return _times(x, s)


def _setup(ctx, inputs, output):
    ctx.s = inputs[1]


tangent_probe = _native._op(tangent_probe, _setup, lambda ctx, d, _: (d * ctx.s, None), direct=True)
tangent_probe_far = _native._op(tangent_probe_far, _setup, lambda ctx, d, _: (d * ctx.s, None))
NAMES = ["tangent_probe", "tangent_probe_far", "tangent_probe_forward"]


@pytest.fixture(params=NAMES)
def probe(request):
    return request.param


@ANYWHERE
def test_a_tangent_is_refused(where, probe):
    x, d = torch.arange(4.0, device=where), torch.ones(4, device=where)
    refused = functools.partial(pytest.raises, NotImplementedError, match=f"gpa::{probe} has no forward-mode")
    for fn in (globals()[probe], getattr(torch.ops.gpa, probe).default):
        def call(t):
            return fn(t, 2.0)[0]
        for leaf in (x, x.clone().requires_grad_()):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(leaf, d)
                with refused():
                    call(dual)
                with refused():
                    fn(s=2.0, x=dual)
                with torch.no_grad(), refused():
                    call(dual)
        for way in (lambda: torch.func.jvp(call, (x,), (d,)), lambda: torch.func.jacfwd(call)(x),
                    lambda: torch.func.vmap(lambda t: torch.func.jvp(call, (t,), (t,)))(x.expand(2, 4)),
                    lambda: torch.func.jvp(torch.func.vmap(call), (x.expand(2, 4),), (x.expand(2, 4),))):
            with refused():
                way()


@ANYWHERE
def test_constants_of_a_forward_derivative_are_taken(where, probe):
    x, d = torch.arange(4.0, device=where), torch.ones(4, device=where)
    for fn in (globals()[probe], getattr(torch.ops.gpa, probe).default):
        with forward_ad.dual_level():
            assert torch.equal(fn(x, 2.0)[0], 2 * x) and fn(x.clone().requires_grad_(), 2.0)[0].requires_grad
            dual = forward_ad.make_dual(x, d)
            assert torch.equal(fn(forward_ad.unpack_dual(dual).primal, 2.0)[0], 2 * x)
            with torch.inference_mode():
                assert torch.equal(fn(torch.ones(3, device=where), 2.0)[0], torch.full((3,), 2.0, device=where))
        y, t = torch.func.jvp(lambda v: 3 * v + fn(x, 2.0)[0], (x,), (d,))
        assert torch.equal(y, 5 * x) and torch.equal(t, 3 * d)
        y, t = torch.func.jvp(lambda v: 3 * v + torch.func.vmap(lambda c: fn(c, 2.0)[0])(x.expand(2, 4))[0], (x,), (d,))
        assert torch.equal(y, 5 * x) and torch.equal(t, 3 * d)


@pytest.mark.gpu
def test_the_operators_refuse_tangents(dev):
    r = lambda *s: torch.randn(*s, device=dev).to(BF)  # noqa: E731
    x, w, heads, at = r(5, 64), r(64, 64), r(1, 2, 5, 64), torch.zeros(5, 2, device=dev, dtype=torch.int32)
    rotary, norm = rotary_axes((16, 16)), r(64)
    _, seen = draft_tree(torch.arange(-1, 4, device=dev, dtype=torch.int32), torch.tensor([3], device=dev, dtype=torch.int32), sizes=None)
    calls = [(lambda t: linear_gate_residual(t, w, activation="silu"), x), (lambda t: linear_gate_residual(x, t), w),
             (lambda t: rotate_heads(t, at, rotary), heads),
             (lambda t: qk_norm_rotate(heads, heads, at, rotary, q_weight=t)[0], norm),
             (lambda t: attention_tree(t, heads, heads, heads, heads, 0.125, seen=seen), heads),
             (lambda t: attention_masked(heads, t, heads, 0.125, causal=True), heads),
             (lambda t: norm_gate_residual(x, t, pre_weight=norm)[0], x)]
    for call, t in calls:
        want = call(t)
        with forward_ad.dual_level():
            assert torch.equal(call(t), want)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward_ad.make_dual(t, t))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (t,), (t,))


@pytest.mark.gpu
def test_a_gradient_with_a_tangent_is_refused(dev):
    """The backward passes over the dispatcher too."""
    r = lambda *s: torch.randn(*s, device=dev).to(BF)  # noqa: E731
    w, rotary, at = r(64, 64), rotary_axes((16, 16)), torch.zeros(5, 2, device=dev, dtype=torch.int32)
    for call, leaf in ((lambda t: linear_gate_residual(t, w), r(5, 64)), (lambda t: rotate_heads(t, at, rotary), r(1, 2, 5, 64))):
        leaf.requires_grad_()
        y = call(leaf)
        d = torch.ones_like(y)
        with forward_ad.dual_level():
            torch.autograd.grad(y, leaf, d, retain_graph=True)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, forward_ad.make_dual(d, d))

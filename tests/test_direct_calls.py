"""Ops whose ordinary eager GPU calls run past the dispatcher: whoever looks on (modes,
transforms, traces, hooks on saved tensors) sees and gets what the registered op gives."""
import functools
from typing import Tuple

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from merging import _native
from merging.fused_attention import attention_tree, draft_tree
from merging.fused_linear import linear_gate_residual
from merging.fused_rotary import qk_norm_rotate, rotary_axes

BF = torch.bfloat16


def direct_probe(x: torch.Tensor, s: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return x * s, x.sum()


def _setup(ctx, inputs, output):
    ctx.s = inputs[1]


direct_probe = _native._op(direct_probe, _setup, lambda ctx, d, _: (d * ctx.s, None), direct=True)


@_native._fake("direct_probe")
def _probe_fake(x, s):
    return x.new_empty(x.shape), x.new_empty(())


@functools.partial(_native._op, direct=True)
def forward_probe(x: torch.Tensor) -> torch.Tensor:
    return x * 2


@_native._fake("forward_probe")
def _forward_fake(x):
    return x.new_empty(x.shape)


@pytest.mark.parametrize("where", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_callable_and_op_agree(where):
    x = torch.arange(4.0, device=where)
    for fn in (direct_probe, torch.ops.gpa.direct_probe.default):
        assert torch.equal(fn(x, 2.0)[0], 2 * x) and not fn(x, 2.0)[0].requires_grad
        assert torch.equal(fn(s=3.0, x=x)[0], 3 * x)
        leaf = x.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(fn(leaf, 2.0)[0].sum(), leaf)[0], torch.full_like(x, 2.0))
        with torch.no_grad():
            assert not fn(leaf, 2.0)[0].requires_grad
        with torch.inference_mode():
            assert fn(x, 2.0)[0].is_inference()
        assert "gpa.direct_probe" in make_fx(lambda t: fn(t, 2.0)[0])(x).code
        assert torch.equal(torch.vmap(lambda t: fn(t, 2.0)[0])(x.expand(3, 4)), (2 * x).expand(3, 4))
        assert torch.equal(torch.compile(lambda t: fn(t, 2.0)[0] + 1, backend="aot_eager", fullgraph=True)(x), 2 * x + 1)
        with FakeTensorMode():
            assert fn(torch.empty(5, device=where), 2.0)[0].shape == (5,)
        assert fn(torch.empty(5, device="meta"), 2.0)[0].is_meta
    out = forward_probe(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no autograd formula"):
        out.sum().backward()


def test_cpu_tensors_are_refused():
    x, heads = torch.zeros(2, 16, dtype=BF), torch.zeros(1, 2, 3, 64, dtype=BF)
    for grad in (False, True):
        with pytest.raises(ValueError, match="GPU tensors"):
            linear_gate_residual(x.clone().requires_grad_(grad), x)
        with pytest.raises(ValueError, match="GPU tensors"):
            qk_norm_rotate(heads.clone().requires_grad_(grad), heads, None, None)
    with pytest.raises(ValueError, match="GPU tensors"):
        draft_tree(torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU tensors"):
        attention_tree(heads, heads, heads, heads, heads, 0.125, seen=torch.zeros(1, 3, 1, dtype=torch.int32))


class _Names(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names = [*getattr(self, "names", []), str(func)]
        return func(*args, **(kwargs or {}))


def _training(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF).requires_grad_()  # noqa: E731
    x, w, b, gate, q_w = r(40, 64), r(256, 64), r(256), r(256), r(64)
    rotary, at = rotary_axes((16, 16)), torch.arange(20, device=dev, dtype=torch.int32)[:, None].expand(20, 2)

    def step():
        y = linear_gate_residual(x, w, b, activation="silu", gate=gate).view(2, 20, 4, 64).transpose(1, 2)
        q, k = qk_norm_rotate(y[:, :2], y[:, 2:], at, rotary, q_weight=q_w, k_weight=q_w)
        return q, k
    return step, [x, w, b, gate, q_w]


@pytest.mark.gpu
def test_modes_see_the_ops(dev):
    step, leaves = _training(dev)
    with _Names() as m:
        q, k = step()
        torch.autograd.grad(q.float().sum() + k.float().sum(), leaves)
    for name in ("linear_gate", "linear_gate_bwd", "head_rotary", "head_rotary_bwd"):
        assert any(n.startswith(f"gpa.{name}.") for n in m.names), (name, m.names)


@pytest.mark.gpu
def test_saved_tensors_that_come_back_from_elsewhere(dev):
    """Kept on the CPU between the passes, as other tensors, and in other strides: the same bits."""
    step, leaves = _training(dev)
    d = [torch.randn(2, 2, 20, 64, device=dev).to(BF) for _ in range(2)]
    want = torch.autograd.grad(step(), leaves, d)
    for hooks in (torch.autograd.graph.save_on_cpu(),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.mT.contiguous().mT if t.dim() > 1 else t)):
        with hooks:
            out = step()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, d), want))


@pytest.mark.gpu
def test_gradients_that_are_expanded_kept_and_differentiated(dev):
    """A sum's gradient has no strides; a graph can be walked twice; there is no second derivative."""
    step, leaves = _training(dev)
    q, k = step()
    total = q.float().sum() + k.float().sum()
    first = torch.autograd.grad(total, leaves, retain_graph=True)
    ones = torch.autograd.grad((q, k), leaves, [torch.ones_like(q), torch.ones_like(k)], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, ones))
    again = torch.autograd.grad(total, leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(again, first))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(again[0].float().sum(), leaves)

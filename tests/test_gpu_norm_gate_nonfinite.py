"""`norm_gate_residual`'s gradients with infinities and NaN in its inputs: they
reach what the definition lets them reach, and change no bit of anything else."""
import math

import pytest
import torch

from merging.fused_norms import norm_gate_residual

pytestmark = pytest.mark.gpu
F, BF = torch.float32, torch.bfloat16
R, C, G = 37, 96, 1
AT = (5, 17)


def _inputs(dev, dt, post, bias, gate, c=C):
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(dt)  # noqa: E731
    t = dict(x=r(R, c), y=r(R, c), w2=r(c), dh=r(R, c), dout=r(R, c), w1=r(c), b1=r(c), b2=r(c), gate=r(c))
    if not post:
        t["w1"] = t["b1"] = None
    if not bias:
        t["b1"] = t["b2"] = None
    if not gate:
        t["gate"] = None
    return t


def _grads(t, kind, use):
    """The gradients by name; `use`: which outputs have one."""
    leaves = {n: t[n].clone().requires_grad_() for n in ("x", "y", "w1", "b1", "gate", "w2", "b2") if t[n] is not None}
    p = {n: leaves.get(n) for n in ("x", "y", "w1", "b1", "gate", "w2", "b2")}
    outs = norm_gate_residual(p["x"], p["y"], p["w2"], post_weight=p["w1"], post_bias=p["b1"], pre_bias=p["b2"],
                              gate=p["gate"], scale=0.5, kind=kind)
    pairs = [(o, t[n]) for o, n in zip(outs, ("dh", "dout")) if n in use]
    got = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])
    return dict(zip(leaves, got))


def _others_keep_their_bits(got, want, col=AT[1], row=None):
    """All but feature `col` (of `row`, where it is a tensor of rows)."""
    for name in want:
        a, b = got[name].clone(), want[name].clone()
        assert a.dim() == 1 or row is not None
        i = (row, col) if a.dim() > 1 else (col,)
        a[i] = b[i] = 0
        assert torch.equal(a, b), name


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("c", [C, 100, 1024])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_one_bad_gradient_without_a_norm_after_the_block(dev, kind, gate, c, bad):
    """dx and dy are elementwise in dh then."""
    t = _inputs(dev, BF, False, True, gate, c)
    for use in (("dh",), ("dh", "dout")):
        want = _grads(t, kind, use)
        dirty = dict(t, dh=t["dh"].clone())
        dirty["dh"][AT] = bad
        got = _grads(dirty, kind, use)
        _others_keep_their_bits(got, want, row=AT[0])
        assert not torch.isfinite(got["x"][AT]) and not torch.isfinite(got["y"][AT])
        if gate:
            one = 0.5 * float(t["y"][AT]) * bad                 # the gate's gradient has it times y
            assert math.isnan(bad) == math.isnan(float(got["gate"][AT[1]]))
            assert math.isnan(bad) or float(got["gate"][AT[1]]) == one


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_products_that_pass_the_range(dev, kind):
    """y dh passes fp32; dy = scale gate dh does not."""
    t = _inputs(dev, BF, False, False, True)
    t["y"], t["dh"] = t["y"] * 1e25, t["dh"] * 1e25
    got = _grads(t, kind, ("dh",))
    assert torch.equal(got["x"], t["dh"])
    want = 0.5 * t["gate"].double() * t["dh"].double()
    # 0.5 gate is exact, its product with dh is rounded to fp32 and to bf16
    assert ((got["y"].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23)).all()


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("name,bad", [("x", math.inf), ("x", math.nan), ("y", math.inf), ("y", math.nan)])
def test_bad_rows_whose_normed_output_has_no_gradient(dev, name, bad, kind, post):
    """Only h's gradient: dx is dh whatever the row holds, the pre-norm's parameters get
    none; dy and the other column sums are what the norm after the block makes of it."""
    t = _inputs(dev, BF, post, True, True)
    want = _grads(t, kind, ("dh",))
    dirty = dict(t, **{name: t[name].clone()})
    dirty[name][AT] = bad
    got = _grads(dirty, kind, ("dh",))
    assert torch.equal(got["x"], t["dh"])
    assert not got["w2"].any() and not got["b2"].any()
    if name == "x":
        assert all(torch.equal(got[n], want[n]) for n in want)
    elif not post:
        _others_keep_their_bits({n: got[n] for n in ("gate",)}, {n: want[n] for n in ("gate",)})
        assert torch.equal(got["y"], want["y"]) and not torch.isfinite(got["gate"][AT[1]])


def test_an_infinite_gradient_of_the_rms_norm(dev):
    """dx = rstd (g - hhat mean(g hhat)): the row's other features are infinite by the
    signs of hhat and of the one product, not NaN."""
    t = _inputs(dev, F, False, False, False)
    t["dout"][AT] = math.inf
    got = _grads(t, "rms", ("dout",))["x"][AT[0]]
    h = (t["x"] + 0.5 * t["y"])[AT[0]]
    want = -h.sign() * (h[AT[1]] * t["w2"][AT[1]]).sign() * math.inf
    keep = torch.arange(C, device=dev) != AT[1]
    assert torch.equal(got[keep], want[keep])
    assert not torch.isfinite(got[AT[1]])

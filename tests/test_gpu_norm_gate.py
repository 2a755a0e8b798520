"""`norm_gate_residual` and its gradients against the definition in 64 bits.

Tolerances: an output is rounded once (half a step u of its type) from fp32
values of rows of C features.  With f = 2^-24: a norm's statistics are off by
at most (C / 64 + 12) f relative (64 lanes' partial sums and a tree), its
result by some more single roundings, all taken together as `e`; where terms
cancel (x + gate u, w t + b, the three terms of a backward row), e counts on the
size of the terms, not of their sum.  Column sums over R rows add (R + 64) f of
their terms' sizes.
"""
import pytest
import torch

from merging import _native
from merging.fused_norms import norm_gate_residual

pytestmark = pytest.mark.gpu
F, BF, HF = torch.float32, torch.bfloat16, torch.float16
f = 2.0 ** -24


def _norm(t, layer, eps):
    mean = t.mean(-1, keepdim=True) if layer else torch.zeros_like(t[..., :1])
    inv = 1 / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (t - mean) * inv, mean, inv


def _norm_back(g, hat, inv, layer):
    """Gradient of t and the size of its terms."""
    c1 = (g * hat).mean(-1, keepdim=True)
    c0 = g.mean(-1, keepdim=True) if layer else torch.zeros_like(c1)
    a1, a0 = (g * hat).abs().mean(-1, keepdim=True), g.abs().mean(-1, keepdim=True)
    return inv * (g - c0 - hat * c1), inv * (g.abs() + a0 + hat.abs() * a1)


def _reference(x, y, w1, b1, gate, w2, b2, scale, layer, eps, gh, gn, u):
    """All in 64 bits: outputs, gradients and their bounds.  gate [G, C]."""
    C, R = x.shape[-1], x.numel() // x.shape[-1]
    z = lambda t: None if t is None else t.double()  # noqa: E731
    x, y, w1, b1, gate, w2, b2, gh, gn = map(z, (x.reshape(R, C), y.reshape(R, C), w1, b1, gate, w2, b2, gh, gn))
    G = 1 if gate is None else gate.shape[0]
    grow = torch.ones(R, C, dtype=torch.float64) if gate is None else gate.repeat_interleave(R // G, 0)
    e = (C / 64 + 40) * f
    yh, my, ry = _norm(y, layer, eps) if w1 is not None else (y, y[:, :1] * 0, y[:, :1] * 0 + 1)
    un = yh * (1 if w1 is None else w1)
    uu = un if b1 is None else un + b1
    # a mean that is large beside the deviations costs its size
    un_e = e * (un.abs() + (my * ry).abs() * (1 if w1 is None else w1.abs()) + (0 if b1 is None else b1.abs()))
    h = x + scale * grow * uu
    h_e = e * x.abs() + (scale * grow).abs() * un_e + e * h.abs() + f * x.abs()
    hh, mh, rh = _norm(h, layer, eps)
    hh_e = rh * h_e + e * hh.abs() + e * (mh * rh).abs() + hh.abs() * (rh * h_e).mean(-1, keepdim=True) \
        + (rh * h_e).mean(-1, keepdim=True)
    out = hh * w2 + (0 if b2 is None else b2)
    got = [(h, u * h.abs() + h_e), (out, u * out.abs() + w2.abs() * hh_e + e * out.abs())]
    if gh is None and gn is None:
        return got
    gh = torch.zeros(R, C, dtype=torch.float64) if gh is None else gh.reshape(R, C)
    gn = torch.zeros(R, C, dtype=torch.float64) if gn is None else gn.reshape(R, C)
    g2 = gn * w2
    back, size = _norm_back(g2, hh, rh, layer)
    # off: the terms' roundings, and what an error of hh does to them
    rel = (hh_e.abs().amax(-1, keepdim=True) / hh.abs().amax(-1, keepdim=True).clamp_min(1e-30))
    d = gh + back
    d_e = e * gh.abs() + (4 * e + 4 * rel) * size
    du = scale * grow * d
    du_e = (scale * grow).abs() * d_e + e * du.abs()
    if w1 is None:
        dy, dy_e = du, du_e
    else:
        g1, g1_e = du * w1, du_e * w1.abs()
        dy, size1 = _norm_back(g1, yh, ry, layer)
        _, size_e = _norm_back(g1_e, yh.abs(), ry, layer)
        rel1 = 4 * e * (1 + (my * ry).abs())
        dy_e = rel1 * size1 + size_e
    cols = lambda t, te: (t.sum(0), te.sum(0) + (R + 64) * f * t.abs().sum(0))  # noqa: E731
    grp = lambda t: t.reshape(G, R // G, C)  # noqa: E731
    got += [(d, u * d.abs() + d_e), (dy, u * dy.abs() + dy_e)]
    if w1 is not None:
        yh_e = e * (yh.abs() + (my * ry).abs())
        got.append(cols(du * yh, du_e * yh.abs() + du.abs() * yh_e))
        if b1 is not None:
            got.append(cols(du, du_e))
    if gate is not None:
        # formed as scale (w1 sum(d yhat) + b1 sum(d))
        t, te = scale * d * uu, abs(scale) * (d_e * (un.abs() + (0 if b1 is None else b1.abs())) + d.abs() * un_e)
        big = abs(scale) * d.abs() * (un.abs() + (0 if b1 is None else b1.abs()))
        got.append((grp(t).sum(1), grp(te).sum(1) + (R // G + 64) * f * grp(big).sum(1)))
    got.append(cols(gn * hh, gn.abs() * hh_e))
    if b2 is not None:
        got.append(cols(gn, gn * 0))
    return got


def _run(dev, shape, dt, pdt=None, layer=False, post=True, bias=False, gate="channel", scale=1.0, which="both",
         mean=0.1, seed=0, stride=0):
    g = torch.Generator().manual_seed(seed)
    pdt = dt if pdt is None else pdt
    C, u = shape[-1], torch.finfo(dt).eps / 2
    r = lambda *s, std=1.0, mid=0.0: torch.randn(*s, generator=g) * std + mid  # noqa: E731
    x, y, gh, gn = (t.to(dt) for t in (r(*shape, std=2.0, mid=mean), r(*shape, std=0.7, mid=-mean), r(*shape), r(*shape)))
    w1, b1, w2, b2 = (t.to(pdt) for t in (r(C, std=0.2, mid=1), r(C, std=0.1), r(C, std=0.2, mid=1), r(C, std=0.1)))
    if not post:
        w1 = None
    if not bias or not post:
        b1 = None
    if not bias:
        b2 = None
    gt = {"none": None, "channel": (C,), "group": (*shape[:1], *(1,) * (len(shape) - 2), C), "full": shape}[gate]
    gt = None if gt is None else r(*gt, std=0.3, mid=0.5).to(pdt)
    if which == "h":
        gn = None
    if which == "out":
        gh = None
    eps = 1e-5
    want = _reference(x, y, w1, b1, None if gt is None else gt.reshape(-1, C), w2, b2, scale, layer, eps, gh, gn, u)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    if stride:                                               # rows of wider tensors
        wide = lambda t: torch.cat((t, t.new_zeros(*shape[:-1], stride)), -1).to(dev)[..., :C]  # noqa: E731
    else:
        wide = to
    X, Y = wide(x), wide(y)
    kw = dict(post_weight=to(w1), post_bias=to(b1), pre_bias=to(b2), gate=to(gt), scale=scale,
              kind="layer" if layer else "rms", eps=eps)
    W2 = to(w2)
    plain = norm_gate_residual(X, Y, W2, **kw)
    leaves = [t for t in (X, Y, kw["post_weight"], kw["post_bias"], kw["gate"], W2, kw["pre_bias"]) if t is not None]
    for t in leaves:
        t.requires_grad_()
    h, out = norm_gate_residual(X, Y, W2, **kw)
    assert torch.equal(h, plain[0]) and torch.equal(out, plain[1]) and h.dtype == dt
    outs = [(t, to(gr)) for t, gr in ((h, gh), (out, gn)) if gr is not None]
    grads = torch.autograd.grad([t for t, _ in outs], leaves, [gr for _, gr in outs], retain_graph=True,
                                allow_unused=True)
    again = torch.autograd.grad([t for t, _ in outs], leaves, [gr for _, gr in outs], allow_unused=True)
    names = ["h", "out", "dx", "dy"] + [n for n, t in (("dw1", w1), ("db1", b1), ("dgate", gt), ("dw2", w2), ("db2", b2))
                                        if t is not None]
    pu = torch.finfo(pdt).eps / 2
    assert len(names) == len(want) == 2 + len(grads)
    for k, (name, got, (ref, bound)) in enumerate(zip(names, [h, out, *grads], want)):
        if k >= 4:
            assert got.dtype == pdt
            bound = bound + pu * ref.abs()
        got = got.detach().cpu().double().reshape(ref.shape)
        slack = 2.0 ** -24 if HF in (dt, pdt) else 1e-30           # fp16's smallest step, halved and doubled
        bad = ~((got - ref).abs() <= bound + slack)
        assert not bad.any(), (name, int(bad.sum()), got[bad][:4], ref[bad][:4], bound[bad][:4])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dt,pdt", [(F, F), (BF, BF), (BF, F), (HF, HF), (HF, F)])
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("C", [8, 512, 520, 1024, 2048, 2056, 4096, 8192])
def test_widths(dev, C, layer, dt, pdt):
    _run(dev, (2, 9, C), dt, pdt, layer=layer, bias=layer, seed=C)


@pytest.mark.parametrize("dt", [F, BF, HF])
@pytest.mark.parametrize("C", [1, 3, 77, 513, 1000, 2047, 4100, 8191])
def test_odd_widths(dev, C, dt):
    """Widths that 8 does not divide."""
    _run(dev, (5, C), dt, layer=C > 1, bias=True, seed=C)


@pytest.mark.parametrize("post,bias,gate", [(False, False, "none"), (False, True, "channel"), (True, False, "none"),
                                            (True, True, "group"), (True, True, "full"), (False, False, "group")])
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("which", ["both", "h", "out"])
def test_parts(dev, which, layer, post, bias, gate):
    _run(dev, (6, 7, 264), BF, layer=layer, post=post, bias=bias, gate=gate, scale=0.7, which=which)
    _run(dev, (3, 2, 5, 1024), HF, F, layer=layer, post=post, bias=bias, gate=gate, scale=-1.3, which=which)


@pytest.mark.parametrize("shape,gate", [((1, 1024), "channel"), ((4099, 512), "channel"), ((3, 1500, 1024), "group"),
                                        ((2500, 3, 128), "group"), ((2300, 2048), "full"), ((1100, 2, 1500), "group"),
                                        ((700, 1, 4096), "group")])
def test_many_rows(dev, shape, gate):
    _run(dev, shape, BF, bias=True, layer=True, gate=gate)


def test_strided_rows(dev):
    _run(dev, (33, 256), BF, stride=64)
    _run(dev, (33, 256), BF, stride=3)                        # rows not 16-byte aligned
    _run(dev, (4, 9, 250), F, stride=2, gate="group")


def test_large_mean(dev):
    """LayerNorm of rows whose mean is 30 times their deviation."""
    _run(dev, (40, 1024), F, layer=True, bias=True, mean=30.0)


def test_empty(dev):
    x = torch.zeros(0, 64, device=dev, dtype=BF, requires_grad=True)
    w = torch.ones(64, device=dev, dtype=BF, requires_grad=True)
    h, out = norm_gate_residual(x, x, w)
    assert h.shape == out.shape == (0, 64)
    g = torch.autograd.grad(out, w, torch.zeros_like(out))[0]
    assert g.shape == (64,) and not g.any()


def test_mixed_parameter_types(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(5, 64, generator=g, device=dev).to(BF)
    w, gate = torch.rand(64, generator=g, device=dev), torch.rand(64, generator=g, device=dev).to(BF)
    gate.requires_grad_()
    a = norm_gate_residual(x, x, w, gate=gate)
    b = norm_gate_residual(x, x, w, gate=gate.float())
    assert torch.equal(a[1], b[1])
    assert torch.autograd.grad(a[1].sum(), gate)[0].dtype == BF


def test_stream_and_graph(dev):
    """Captured forward and backward, replayed on new inputs between eager calls."""
    g = torch.Generator(device=dev).manual_seed(3)
    make = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)  # noqa: E731
    x, y, gate, w1, w2 = (t.requires_grad_() for t in (make(2, 70, 1024), make(2, 70, 1024), make(2, 1, 1024),
                                                       make(1024), make(1024)))
    gh, gn = make(2, 70, 1024), make(2, 70, 1024)

    def step():
        out = norm_gate_residual(x, y, w2, post_weight=w1, gate=gate)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (x, y, gate, w1, w2), (gh, gn))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        with torch.no_grad():
            for t in (x, y, gate, w1, w2):
                t.copy_(make(*t.shape))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), turn


def test_reference_by_differences(dev):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).double()  # noqa: E731
    for layer in (False, True):
        t = [r(6, 5), r(6, 5), r(5), r(5), r(2, 5), r(5), r(5)]           # x y w1 b1 gate w2 b2
        gh, gn = r(6, 5), r(6, 5)
        call = lambda a=None, b=None: _reference(*t, 0.7, layer, 1e-5, a, b, 0.0)  # noqa: E731

        def loss():
            h, out = (v for v, _ in call())
            return (h * gh).sum() + (out * gn).sum()
        for leaf, (want, _) in zip(t, call(gh, gn)[2:]):
            for at in (0, leaf.numel() - 1):
                flat, eps = leaf.view(-1), 1e-6
                flat[at] += eps
                up = loss()
                flat[at] -= 2 * eps
                down = loss()
                flat[at] += eps
                assert abs((up - down) / (2 * eps) - want.reshape(-1)[at]) < 1e-6 * (1 + abs(want.reshape(-1)[at]))


def test_op_checks(dev):
    x = torch.randn(3, 4, 64, device=dev, dtype=BF, requires_grad=True)
    # one leaf a place: the sum of three bf16 gradients of one leaf goes by their order
    y = torch.randn(3, 4, 64, device=dev, dtype=BF, requires_grad=True)
    w, w1, b1 = (torch.randn(64, device=dev, dtype=BF, requires_grad=True) for _ in range(3))
    gate = torch.randn(3, 64, device=dev, dtype=BF, requires_grad=True)
    torch.library.opcheck(torch.ops.gpa.norm_gate.default, (x, y, w1, b1, gate, w, None, 0.5, True, 1e-5, True))
    d, wd = x.detach(), w.detach()
    stats = _native.norm_gate(d, d, wd, None, None, wd, None, 1.0, False, 1e-5, True)[2]
    torch.library.opcheck(torch.ops.gpa.norm_gate_bwd.default,
                          (d, None, d, d, wd, None, None, wd, None, stats, 1.0, False))

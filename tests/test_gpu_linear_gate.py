"""`linear_gate_residual` and its gradients against the definition in 64 bits.

Tolerances, with f = 2^-24 and u half a step of the tensors' type (tiny: half the smallest
step of fp16): a sum over K products of 16-bit values, exact in fp32, is off by at most
(K + 16) f of their sizes.  GELU's distribution is off by 1e-7 (its formula's 7.5e-8 and
roundings) + 16 f, a logistic value s of t by s (1 - s) (|t| + 4) 4 f + 4 f s, and what
comes in off moves an activation by at most 1.13 of it and its slope by 1.2 (GELU's
second derivative is below 0.8, its tanh form's below 1, SiLU's 0.5; ReLU's slope is open
where the sum's sign is); without a gate a bf16 call's slopes come from sums kept in fp16.  dz is rounded once (fp16 with a gate: after a scaling that makes
the gate's largest value one or more), sums over R rows add (R + 64) f of their terms.
"""
import math

import pytest
import torch

from merging import _native
from merging.fused_linear import linear_gate_residual

pytestmark = pytest.mark.gpu
F, BF, HF = torch.float32, torch.bfloat16, torch.float16
f = 2.0 ** -24


def _act(z, name):
    """(act, slope, act's own error, slope's own error) in 64 bits."""
    if name is None:
        return z, torch.ones_like(z), z * 0, z * 0
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), z * 0, z * 0
    if name == "gelu":
        s = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        d = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        off = 1e-7 + 16 * f
        return z * s, s + z * d, z.abs() * off + 2 * f * (z * s).abs(), off + z.abs() * d * (z * z + 8) * 2 * f + 4 * f
    t = z if name == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    dt = z if name == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 3 * 0.044715 * z ** 3)
    s = torch.sigmoid(t)
    off = s * (1 - s) * (t.abs() + 4) * 4 * f + 4 * f * s
    return z * s, s + dt * s * (1 - s), z.abs() * off + 2 * f * (z * s).abs(), off * (1 + dt.abs()) + 8 * f * (1 + (dt * s * (1 - s)).abs())


def _reference(x, w, bias, gate, residual, act, dy, u, tiny):
    """[(value, bound)] of y and, with dy, of the gradients of what is there."""
    x, w, bias, gate, residual, dy = (None if t is None else t.double() for t in (x, w, bias, gate, residual, dy))
    (M, K), N = x.shape, w.shape[0]
    z = x @ w.t() + (0 if bias is None else bias)
    ze = (K + 16) * f * (x.abs() @ w.abs().t() + (0 if bias is None else bias.abs()))
    a, slope, ae, se = _act(z, act)
    ae = ae + 1.13 * ze
    g = torch.ones(N, dtype=torch.float64, device=x.device) if gate is None else gate
    y = a * g + (0 if residual is None else residual)
    got = [(y, u * y.abs() + ae * g.abs() + 4 * f * ((a * g).abs() + y.abs()) + tiny)]
    if dy is None:
        return got
    kept = u == 2.0 ** -8 and gate is None and act        # z is kept in fp16
    se = se + 1.2 * (ze + (2.0 ** -11 * z.abs() + 2.0 ** -25 if kept else 0)) + (((z.abs() <= ze) & (ze > 0)).double() if act == "relu" else 0)
    dz = dy * g * slope
    off = (dy * g).abs() * se + 4 * f * dz.abs() if act or gate is not None else dz * 0
    least = tiny * g.abs().max() if gate is not None else tiny
    rounded = off + ((u * (dz.abs() + off) + least) if act or gate is not None else 0)
    dx, dw = dz @ w, dz.t() @ x
    got.append((dx, u * dx.abs() + rounded @ w.abs() + (N + 16) * f * (dz.abs() @ w.abs()) + tiny))
    got.append((dw, u * dw.abs() + rounded.t() @ x.abs() + (M + 16) * f * (dz.abs().t() @ x.abs()) + tiny))
    if bias is not None:
        got.append((dz.sum(0), off.sum(0) + (M + 64) * f * dz.abs().sum(0)))
    if gate is not None:
        got.append(((dy * a).sum(0), (dy.abs() * ae).sum(0) + (M + 64) * f * (dy * a).abs().sum(0)))
    if residual is not None:
        got.append((dy, dy * 0))
    return got


def _check(dev, M, N, K, dt=BF, pdt=None, act=None, bias=True, gate=False, residual=False, grad=True, layout="plain",
           gate_size=0.4, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    pdt = dt if pdt is None else pdt
    u, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == HF else 0.0
    r = lambda *s, std=1.0, mid=0.0: torch.randn(*s, generator=g, device=dev) * std + mid  # noqa: E731

    def laid(t):
        if layout == "wide":                                 # columns of a wider tensor
            return torch.nn.functional.pad(t, (8, 16))[:, 8:-16] if t.shape[0] else t
        if layout == "odd":
            return torch.nn.functional.pad(t, (3, 2))[:, 3:-2]
        return t.t().contiguous().t() if layout == "turned" else t
    x, w = laid(r(M, K, std=1.1).to(dt)), laid(r(N, K, std=max(K, 1) ** -0.5 * 1.5).to(dt))
    b = r(N, std=0.3).to(pdt) if bias else None
    gt = r(N, std=0.5 * gate_size, mid=gate_size).to(pdt) if gate else None
    res = laid(r(M, N, std=2.0).to(dt)) if residual else None
    dy = laid(r(M, N).to(dt)) if grad else None
    want = _reference(x, w, b, gt, res, act, dy, u, tiny)
    leaves = [t.detach().requires_grad_(grad) for t in (x, w, b, gt, res) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b, gt, res)]
    call = lambda: linear_gate_residual(args[0], args[1], args[2], activation=act, gate=args[3], residual=args[4])  # noqa: E731
    y = call()
    assert y.shape == (M, N) and y.dtype == dt
    got = [y.detach()]
    if grad:
        got += torch.autograd.grad(y, leaves, dy)
        again = torch.autograd.grad(call(), leaves, dy)
        assert all(torch.equal(a, c) for a, c in zip(got[1:], again)), "two backward passes differ"
    else:
        assert torch.equal(call(), y)
    names = ["y", "dx", "dw"] + [n for n, t in (("dbias", b), ("dgate", gt), ("dresidual", res)) if t is not None]
    for name, a, (value, bound) in zip(names, got, want):
        if name in ("dbias", "dgate"):
            pu = torch.finfo(pdt).eps / 2
            bound = bound + pu * (value.abs() + bound) + (2.0 ** -25 if pdt == HF else 0)
        bad = ~((a.double() - value).abs() <= bound + 1e-37)
        assert a.shape == value.shape and not bad.any(), \
            f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((a.double() - value).abs() / (bound + 1e-37)).max()):.3g} bounds"
    assert len(names) == len(got) or not grad


SIZES = [(1, 16, 8), (1, 1, 1), (3, 5, 7), (8, 4096, 4096), (16, 100, 1000), (17, 33, 40), (33, 1000, 520), (64, 17, 2056),
         (65, 64, 64), (66, 7, 9), (100, 200, 300), (129, 257, 72), (1374, 1001, 777), (1000, 24, 4096), (24, 1000, 4096),
         (2000, 1024, 1024), (5000, 264, 136), (300, 3000, 31), (2111, 2113, 40), (70, 70, 8000), (4099, 8, 8)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(dev, dt, M, N, K):
    _check(dev, M, N, K, dt=dt, act="silu", gate=True, residual=True)
    _check(dev, M, N, K, dt=dt, bias=False)


@pytest.mark.parametrize("M,N,K", [(8192, 4096, 512), (10_992, 1024, 264), (4096, 4096, 4096), (5000, 5000, 104), (3000, 8000, 1000),
                                   (20_000, 2000, 200)])
def test_large_products(dev, M, N, K):
    _check(dev, M, N, K, act="gelu_tanh")


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kw", [dict(), dict(gate=True), dict(residual=True, bias=False), dict(gate=True, residual=True, pdt=F),
                                dict(bias=False, gate=True, grad=False)])
def test_options(dev, act, dt, kw):
    _check(dev, 200, 136, 96, dt=dt, act=act, **kw)
    _check(dev, 9, 50, 72, dt=dt, act=act, **kw)


@pytest.mark.parametrize("layout", ["wide", "odd", "turned"])
@pytest.mark.parametrize("M,N,K", [(300, 264, 128), (5, 40, 64), (300, 263, 127)])
def test_layouts(dev, layout, M, N, K):
    _check(dev, M, N, K, act="gelu", gate=True, residual=True, layout=layout)
    _check(dev, M, N, K, layout=layout, residual=True)


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("gate_size", [1e-5, 1e-7, 300.0])
def test_gates_out_of_fp16s_middle(dev, act, gate_size):
    """dz in fp16 keeps its accuracy under gates at the format's ends."""
    _check(dev, 150, 64, 80, dt=HF, pdt=F, act=act, gate=True, gate_size=gate_size)


@pytest.mark.parametrize("gate_size", [0.95, 1.05, 1e-5])
def test_gradients_near_fp16s_largest(dev, gate_size):
    """dz of a gradient of 50,000 stays in range inside (1.13 times it at most), and dx with it: x's
    gradient is dy gate w of one output, off by half a step for dz, w's product being exact, and for
    itself (2 * 2^-11 of its value, and as much again for the product of both)."""
    dy = torch.tensor([[50_000.0], [-49_000.0], [3.0]], device=dev, dtype=HF).repeat(20, 1)
    x = torch.ones(60, 8, device=dev, dtype=HF, requires_grad=True)
    w = torch.full((1, 8), 0.125, device=dev, dtype=HF)
    gate = torch.tensor([gate_size], device=dev)
    y = linear_gate_residual(x, w, gate=gate, activation="relu")
    dx, = torch.autograd.grad(y, x, dy)
    want = (dy.double() * gate.double() * 0.125).expand(-1, 8)
    assert ((dx.double() - want).abs() <= want.abs() * (2.0 ** -10 + 2.0 ** -21) + 2.0 ** -25).all()


@pytest.mark.parametrize("tile,M,N,K", [(0, 4096, 4096, 4096), (1, 8192, 2048, 1024), (2, 2048, 2048, 1024), (3, 700, 520, 256)])
def test_every_tile_and_layout(dev, tile, M, N, K):
    """Sizes of each kind of tile, forward and (dx, dw) turned, with edges in both directions."""
    _check(dev, M, N, K, act="relu", bias=False)
    _check(dev, M - 8 - tile, N - 24, K - 8, dt=HF)


def test_batched_shapes_and_casts(dev):
    """Leading dimensions, fp32 x (cast to bf16, or the autocast dtype), parameters of mixed types."""
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, w, b, res = r(2, 3, 50, 64), r(40, 64), r(40), r(2, 3, 50, 40)
    y = linear_gate_residual(x, w, b, residual=res, activation="gelu")
    assert y.shape == res.shape and y.dtype == BF
    flat = linear_gate_residual(x.to(BF).view(-1, 64), w.to(BF), b, residual=res.to(BF).view(-1, 40), activation="gelu")
    assert torch.equal(y.view(-1, 40), flat)
    with torch.autocast("cuda", dtype=HF):
        assert linear_gate_residual(x, w, b).dtype == HF
    one = linear_gate_residual(x[0, 0, 0].to(BF), w.to(BF), b.to(BF))
    assert one.shape == (40,)
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(linear_gate_residual(x, w, b, gate=b.to(BF)).float().sum(), (x, w))
    assert dx.dtype == F and dx.shape == x.shape and dw.dtype == F


def test_gradients_that_are_not_wanted(dev):
    """Each gradient alone is the one that comes with the others."""
    g = torch.Generator(device=dev).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)  # noqa: E731
    ts, dy = [r(130, 64), r(72, 64), r(72), r(72), r(130, 72)], r(130, 72)

    def grads(which):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate(ts)]
        y = linear_gate_residual(leaves[0], leaves[1], leaves[2], gate=leaves[3], residual=leaves[4], activation="silu")
        return torch.autograd.grad(y, [leaves[i] for i in which], dy)
    every = grads(range(5))
    for i in range(5):
        assert torch.equal(grads([i])[0], every[i])


def test_gradients_against_differences(dev):
    """y's change along a direction of all fp32-held inputs of 64-bit sums: fp16 inputs on a
    grid of 1/16, so that x +- h d is exact; the difference of y in 64 bits is the
    definition's, the gradients the kernel's."""
    g = torch.Generator(device=dev).manual_seed(4)
    grid = lambda *s: torch.round(torch.randn(*s, generator=g, device=dev) * 16) / 16  # noqa: E731
    ts = [grid(40, 24), grid(16, 24) / 4, grid(16), grid(16), grid(40, 16)]
    dirs, dy = [grid(*t.shape) for t in ts], grid(40, 16)

    def value(ts):
        x, w, b, gt, res = (t.double() for t in ts)
        z = x @ w.t() + b
        return ((res + gt * z * torch.sigmoid(z)) * dy.double()).sum()
    leaves = [t.to(HF).requires_grad_() for t in ts]
    y = linear_gate_residual(leaves[0], leaves[1], leaves[2], gate=leaves[3], residual=leaves[4], activation="silu")
    grads = torch.autograd.grad(y, leaves, dy.to(HF))
    along = sum((a.double() * d.double()).sum() for a, d in zip(grads, dirs))
    size = sum((a.double() * d.double()).abs().sum() for a, d in zip(grads, dirs))
    h = 2.0 ** -10
    diff = (value([t + h * d for t, d in zip(ts, dirs)]) - value([t - h * d for t, d in zip(ts, dirs)])) / (2 * h)
    assert abs(float(along - diff)) <= 3 * 2.0 ** -11 * float(size)


def test_infinities_stay_in_their_row_and_column(dev):
    r = lambda *s: torch.randn(*s, device=dev).to(BF)  # noqa: E731
    for M in (20, 300):
        x, w, res = r(M, 64), r(80, 64), r(M, 80)
        x2, res2 = x.clone(), res.clone()
        x2[3, 5], res2[7, 9] = math.inf, math.nan
        for act in (None, "gelu", "gelu_tanh", "silu", "relu"):
            a, b = (linear_gate_residual(p, w, activation=act, residual=q) for p, q in ((x, res), (x2, res2)))
            same = torch.ones_like(a, dtype=torch.bool)
            same[3], same[7, 9] = False, False
            assert torch.equal(a[same], b[same]) and b[7, 9].isnan() and not torch.isnan(b[3]).any()
            lo = w[:, 5] < 0
            assert (b[3][~lo] == math.inf).all()
            assert torch.equal(b[3][lo], res[3][lo]) if act else (b[3][lo] == -math.inf).all()


def test_empty(dev):
    for M, N, K in ((0, 8, 16), (5, 0, 16), (5, 8, 0), (100, 8, 0)):
        x, w = torch.zeros(M, K, device=dev, dtype=BF), torch.zeros(N, K, device=dev, dtype=BF)
        b = torch.arange(N, device=dev).to(BF)
        for t in (x, w, b):
            t.requires_grad_()
        y = linear_gate_residual(x, w, b, activation="relu")
        assert torch.equal(y, b.detach().expand(M, N))
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert not dx.any() and not dw.any() and torch.equal(db, torch.tensor(M, device=dev).to(BF) * (b.detach() > 0))


def test_captured_and_replayed(dev):
    """Forward and backward in a graph, replayed with new values, eager calls between."""
    r = lambda *s: torch.randn(*s, device=dev).to(BF)  # noqa: E731
    for M in (4, 400):
        x, w, b, res, dy = r(M, 512), r(136, 512) * 0.05, r(136), r(M, 136), r(M, 136)

        def step():
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = linear_gate_residual(*leaves, activation="gelu", residual=res)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i in range(3):
            x.normal_(), dy.normal_()
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_on_another_stream(dev):
    r = lambda *s: torch.randn(*s, device=dev).to(BF)  # noqa: E731
    x, w = r(500, 4096), r(64, 4096)
    want, side = linear_gate_residual(x, w), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_gate_residual(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_registration(dev):
    r = lambda *s: torch.randn(*s, device=dev).to(BF).requires_grad_()  # noqa: E731
    torch.library.opcheck(torch.ops.gpa.linear_gate.default, (r(70, 16), r(24, 16), r(24), r(24), r(70, 24), 3, True))
    torch.library.opcheck(torch.ops.gpa.linear_gate.default, (r(5, 16).detach(), r(24, 16).detach(), None, None, None, 0, False))
    assert _native.linear_gate(r(5, 16).detach(), r(24, 16).detach(), None, None, None, 0, False)[1].numel() == 0

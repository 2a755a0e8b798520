"""`qk_norm_rotate` and `rotate_heads` and their gradients against the definition in
64 bits.

Tolerances, with f = 2^-24 and u half a step of the outputs' type (plus half the
smallest step of fp16, 2^-25): a norm's statistics and result are off by e = (D / 64 +
40) f of their terms (partial sums of 8 pairs a lane, a tree, single roundings).
An angle is formed in 64 bits (off by 2^-50 of itself, 2^-51 for three roundings
and one of the table) and rounded to fp32 in turns below one half (2^-26 turns, 1.6
f radians); sine and cosine add 4 f: a rotated value is off by r = 10 f plus the
angle's 2^-50 t of |a| + |b|.  Sums over R rows add (R + 64) f of their terms' sizes.
"""
import math

import pytest
import torch

from merging import _native
from merging.fused_rotary import RotaryAxes, qk_norm_rotate, rotary_axes, rotate_heads

pytestmark = pytest.mark.gpu
F, BF, HF = torch.float32, torch.bfloat16, torch.float16
f = 2.0 ** -24


def _features(sections, pairing):
    """(first feature, second feature, axis) of every pair."""
    total, at, out = sum(sections), 0, []
    for a, n in enumerate(sections):
        for i in range(n):
            j = at + i
            out.append({"half": (j, total + j), "interleaved": (2 * j, 2 * j + 1),
                        "blocks": (2 * at + i, 2 * at + n + i)}[pairing] + (a,))
        at += n
    return out


def _turn(x, t, pairs, err, back=False):
    """x [B, H, N, D] in 64 bits turned by t [B, N, pairs], and its bound; err: x's own."""
    if not pairs:
        return x.clone(), err.clone()
    a, b = (torch.tensor(p) for p in list(zip(*pairs))[:2])
    c, s = torch.cos(t)[:, None], torch.sin(t)[:, None] * (-1 if back else 1)
    y, e = x.clone(), err.clone()
    xa, xb, r = x[..., a], x[..., b], 10 * f + 2.0 ** -50 * t.abs()[:, None]
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    both, own = xa.abs() + xb.abs(), err[..., a] * 1.0
    e[..., a] = err[..., a] * c.abs() + err[..., b] * s.abs() + r * both
    e[..., b] = err[..., b] * c.abs() + own * s.abs() + r * both
    return y, e


def _reference(x, w, b, t, pairs, kind, eps, dy, u, tiny):
    """Everything for one tensor [B, H, N, D]: [(value, bound)] of y, and with dy of dx, dw, db."""
    x, w, b, dy = (None if v is None else v.double() for v in (x, w, b, dy))
    D, R = x.shape[-1], x.numel() // x.shape[-1]
    e = (D / 64 + 40) * f
    ones = torch.ones(D, dtype=torch.float64)
    if kind is None:
        n, ne, hat = x, x * 0, None
    else:
        mean = x.mean(-1, keepdim=True) if kind == "layer" else x[..., :1] * 0
        inv = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
        hat = (x - mean) * inv
        he = e * (hat.abs() + (mean * inv).abs() * 2)
        ww = ones if w is None else w
        n = hat * ww + (0 if b is None else b)
        ne = he * ww.abs() + 2 * f * (hat * ww).abs() + f * n.abs()
    y, ye = _turn(n, t, pairs, ne)
    got = [(y, u * y.abs() + ye + tiny)]
    if dy is None:
        return got
    dn, de = _turn(dy, t, pairs, dy * 0, back=True)
    if kind is None:
        return got + [(dn, u * dn.abs() + de + tiny)]
    g, ge = dn * ww, de * ww.abs() + f * (dn * ww).abs()
    c1, c0 = (g * hat).mean(-1, keepdim=True), g.mean(-1, keepdim=True) if kind == "layer" else g[..., :1] * 0
    a1, a0 = (g * hat).abs().mean(-1, keepdim=True), g.abs().mean(-1, keepdim=True) if kind == "layer" else c0
    dx = inv * (g - c0 - hat * c1)
    size = inv * (g.abs() + a0 + hat.abs() * a1)
    off1 = (ge * hat.abs() + g.abs() * he).mean(-1, keepdim=True)
    off = inv * (ge + (ge.mean(-1, keepdim=True) if kind == "layer" else 0) + hat.abs() * off1 + he * a1)
    got.append((dx, u * dx.abs() + off + 2 * e * size + tiny))
    rows = lambda v, ve: (v.sum((0, 1, 2)), ve.sum((0, 1, 2)) + (R + 64) * f * v.abs().sum((0, 1, 2)))  # noqa: E731
    if w is not None:
        got.append(rows(dn * hat, de * hat.abs() + dn.abs() * he))
    if b is not None:
        got.append(rows(dn, de))
    return got


def _near(name, got, want, bound, rounded=None):
    got = got.detach().double().cpu()
    if rounded is not None:                       # a parameter's gradient is rounded to its type
        bound = bound + torch.finfo(rounded).eps / 2 * (want.abs() + bound) + (2.0 ** -25 if rounded == HF else 0)
    bad = ~((got - want).abs() <= bound)
    assert got.shape == want.shape and not bad.any(), \
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound).max()):.3g} bounds"


def _check(dev, B=2, H=3, Hk=2, N=5, D=64, dt=BF, pdt=None, kind="rms", weights=True, biases=None, sections=(32,),
           pairing="half", ladder="shared", order="sections", positions="far", pos_dt=torch.int32, base=10000.0,
           grad=True, eps=1e-6, layout="bnhd", seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    pdt = dt if pdt is None else pdt
    u, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == HF else 0.0
    r = lambda *s, std=1.0, mid=0.0: torch.randn(*s, generator=g) * std + mid  # noqa: E731
    biases = kind == "layer" if biases is None else biases

    def laid(heads):
        x = r(B, N, heads, D, std=1.5, mid=mean).to(dt)
        if layout == "bnhd":                      # a slice of a wider projection
            wide = torch.zeros(B, N, heads + 3, D, dtype=dt, device=dev)
            wide[:, :, 1:heads + 1] = x.to(dev)
            return wide[:, :, 1:heads + 1].transpose(1, 2)
        if layout == "bhnd":
            return x.to(dev).transpose(1, 2).contiguous()
        if layout == "odd":                       # rows that are not 16-byte aligned
            wide = torch.zeros(B, N, heads, D + 1, dtype=dt, device=dev)
            wide[..., 1:] = x.to(dev)
            return wide[..., 1:].transpose(1, 2)
        return x.to(dev).permute(0, 2, 3, 1).contiguous().transpose(2, 3)   # features apart
    q, k = laid(H), laid(Hk) if Hk else None
    A = len(sections)
    shape = (B, N, A) if positions != "shared" else (N, A)
    lo, hi = {"far": (-4_000_000, 4_000_000), "near": (0, 50), "shared": (0, 3000)}[positions]
    p = torch.randint(lo, hi, shape, generator=g).to(pos_dt)
    if pos_dt == F:
        p = p + 0.37
    rot = None
    pairs, t = [], torch.zeros(B, N, 0, dtype=torch.float64)
    if sum(sections):
        rot = rotary_axes(sections, base=base, ladder=ladder, pairing=pairing, order=order, device=dev)
        pairs = _features(sections, pairing)
        ax = torch.tensor([x[2] for x in pairs]) if order == "sections" else rot.axes.cpu().long()
        own, cnt = [], {}
        for j, a in enumerate(ax.tolist()):
            i = cnt.get(a, 0)
            cnt[a] = i + 1
            own.append(base ** (-(i / sections[a]) if ladder == "own" else -(j / sum(sections))))
        t = p.double().expand(B, N, A)[..., ax] * torch.tensor(own, dtype=torch.float64)
    par = [r(D, std=0.3, mid=1.0).to(pdt) if weights and kind else None for _ in range(2)]
    par += [r(D, std=0.2).to(pdt) if biases and kind else None for _ in range(2)]
    dpar = [None if v is None else v.to(dev).requires_grad_(grad) for v in par]
    q.requires_grad_(grad)
    if k is not None:
        k.requires_grad_(grad)
    pd = p.to(dev) if rot is not None else None
    if kind is None:
        assert k is None
        out = [rotate_heads(q, pd, rot)]
    else:
        out = list(qk_norm_rotate(q, k, pd, rot, q_weight=dpar[0], k_weight=dpar[1], q_bias=dpar[2], k_bias=dpar[3],
                                  kind=kind, eps=eps))
    for o, x in zip(out, (q, k)):
        assert o.shape == x.shape and o.dtype == dt and o.stride(-1) == 1
    dys = [r(*o.shape).to(dt) for o in out]
    leaves = [v for v in (q, k, *dpar) if v is not None]
    grads = {}
    if grad:
        got = torch.autograd.grad(out, leaves, [d.to(dev) for d in dys])
        grads = {id(v): gr for v, gr in zip(leaves, got)}
        again = torch.autograd.grad(
            [rotate_heads(q, pd, rot)] if kind is None else
            list(qk_norm_rotate(q, k, pd, rot, q_weight=dpar[0], k_weight=dpar[1], q_bias=dpar[2], k_bias=dpar[3],
                                kind=kind, eps=eps)), leaves, [d.to(dev) for d in dys])
        assert all(torch.equal(a, b) for a, b in zip(got, again)), "two backward passes differ"
    for i, (x, o) in enumerate(zip((q, k), out)):
        want = _reference(x.detach().cpu(), par[i], par[2 + i], t, pairs, kind, eps, dys[i] if grad else None, u, tiny)
        _near("qk"[i], o, *want[0])
        if not grad:
            continue
        _near("d" + "qk"[i], grads[id(x)], *want[1])
        assert grads[id(x)].dtype == dt
        rest = want[2:]
        for name, v in (("w", dpar[i]), ("b", dpar[2 + i])):
            if v is not None:
                _near("d" + "qk"[i] + "_" + name, grads[id(v)], *rest.pop(0), rounded=pdt)


@pytest.mark.parametrize("dt", [BF, HF, F])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("D,sections,pairing", [(64, (8, 12, 12), "half"), (128, (64,), "interleaved"),
                                                (64, (16, 16), "blocks"), (256, (128,), "half")])
def test_norm_and_rotation(dev, dt, kind, D, sections, pairing):
    _check(dev, D=D, dt=dt, kind=kind, sections=sections, pairing=pairing)


@pytest.mark.parametrize("dt", [BF, HF, F])
@pytest.mark.parametrize("D,sections,pairing", [
    (2, (1,), "half"), (2, (0,), "half"), (6, (1, 1), "interleaved"), (10, (3, 0, 2), "blocks"), (34, (17,), "half"),
    (66, (9, 3, 5, 8, 2, 1, 3, 1), "blocks"), (96, (20, 14), "blocks"), (254, (100,), "interleaved"),
    (126, (31,), "half"), (80, (16, 24), "half"), (80, (40,), "interleaved"), (256, (16,) * 8, "blocks"),
    (256, (1, 13, 13, 13, 13, 13, 13, 13), "blocks"), (64, (8, 8), "interleaved"), (72, (36,), "half")])
def test_head_dims_and_sections(dev, dt, D, sections, pairing):
    _check(dev, D=D, dt=dt, sections=sections, pairing=pairing, kind="layer")
    _check(dev, D=D, dt=dt, sections=sections, pairing=pairing, kind=None, Hk=0) if sum(sections) else None


@pytest.mark.parametrize("layout", ["bnhd", "bhnd", "odd", "apart"])
@pytest.mark.parametrize("dt", [BF, F])
@pytest.mark.parametrize("pairing", ["half", "interleaved"])
def test_layouts(dev, layout, dt, pairing):
    _check(dev, layout=layout, dt=dt, pairing=pairing, sections=(20, 12))
    _check(dev, layout=layout, dt=dt, pairing=pairing, sections=(32,), kind=None, Hk=0)


@pytest.mark.parametrize("B,H,Hk,N,D", [
    (1, 1, 1, 1, 64), (8, 16, 4, 1, 128), (1, 1, 0, 7, 64), (1, 1, 1, 4099, 64), (2, 5, 1, 1374, 64), (1, 40, 8, 700, 128),
    (1, 2, 2, 9001, 64), (3, 64, 1, 33, 32), (1, 3, 7, 2049, 16), (1, 300, 200, 3, 64), (1, 16, 16, 3000, 64), (40, 1, 2, 31, 256)])
def test_sizes(dev, B, H, Hk, N, D):
    _check(dev, B=B, H=H, Hk=Hk, N=N, D=D, sections=(D // 2,), kind="rms" if Hk else None)


@pytest.mark.parametrize("kw", [
    dict(weights=False), dict(weights=False, biases=True), dict(kind="rms", biases=True), dict(kind="layer", biases=False),
    dict(pdt=F), dict(pdt=F, kind="layer", dt=HF), dict(sections=(0,)), dict(sections=(0, 0, 32)), dict(order="dealt", sections=(10, 11, 11)),
    dict(order="dealt", ladder="own", sections=(4, 9, 1), pairing="interleaved"), dict(ladder="own", sections=(12, 20)),
    dict(positions="shared"), dict(pos_dt=torch.int64), dict(pos_dt=F, positions="near"), dict(base=2.5), dict(eps=0.0),
    dict(eps=1.0), dict(kind="layer", mean=30.0, dt=F), dict(grad=False), dict(seed=5, kind="layer")])
def test_options(dev, kw):
    _check(dev, **kw)


def test_positions_of_wide_integers(dev):
    """int64 positions that int32 does not hold, against angles in 64 bits."""
    rot = rotary_axes((4,), base=1000.0, device=dev)
    x = torch.randn(1, 1, 3, 8, generator=torch.Generator().manual_seed(1))
    p = torch.tensor([[2 ** 40], [-2 ** 33 - 1], [7]])
    y = rotate_heads(x.to(dev), p.to(dev), rot)
    t = (p.double() * rot.freqs.cpu())[None]
    want, bound = _turn(x.double(), t, _features((4,), "half"), torch.zeros_like(x).double())
    _near("y", y, want, bound + f * want.abs())


@pytest.mark.parametrize("dt", [BF, F])
def test_gradients_of_one_output_alone(dev, dt):
    """The loss reads q or k alone: the other's gradients are absent."""
    g = torch.Generator().manual_seed(3)
    rot = rotary_axes((32,), device=dev)
    for one in (0, 1):
        x = [torch.randn(1, 2, 9, 64, generator=g).to(dt).to(dev).requires_grad_() for _ in range(2)]
        w = [torch.randn(64, generator=g).to(dt).to(dev).requires_grad_() for _ in range(2)]
        p = torch.arange(9, device=dev)[:, None]
        out = qk_norm_rotate(*x, p, rot, q_weight=w[0], k_weight=w[1])
        dy = torch.randn(1, 2, 9, 64, generator=g).to(dt).to(dev)
        got = torch.autograd.grad(out[one], x + w, dy, allow_unused=True)
        both = torch.autograd.grad(qk_norm_rotate(*x, p, rot, q_weight=w[0], k_weight=w[1]), x + w, [dy, dy])
        for i in range(4):
            if i % 2 == one:
                # the sums' partials are cut otherwise: equal but for their order
                if i < 2:
                    assert torch.equal(got[i], both[i])
                else:
                    assert torch.allclose(got[i].float(), both[i].float(), rtol=2 * torch.finfo(dt).eps, atol=1e-4)
            else:
                assert got[i] is None or not got[i].any()


def test_gradients_against_differences(dev):
    """fp32: (L(x + h d) - L(x - h d)) / 2h along a random direction of all inputs.  The
    truncation h^2 / 6 of the third derivative and the roundings, 2^-22 of the terms'
    sum over h, stay below 1e-3 of a derivative of order 10."""
    g = torch.Generator().manual_seed(11)
    rot = rotary_axes((5, 7), ladder="own", pairing="blocks", device=dev)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    leaves = [r(2, 3, 6, 32), r(2, 1, 6, 32), r(32), r(32), r(32), r(32)]
    p, cq, ck = torch.randint(0, 9, (2, 6, 2), generator=g).to(dev), r(2, 3, 6, 32), r(2, 1, 6, 32)
    dirs = [r(*t.shape) for t in leaves]

    def loss(ts):
        q, k = qk_norm_rotate(ts[0], ts[1], p, rot, q_weight=ts[2], k_weight=ts[3], q_bias=ts[4], k_bias=ts[5],
                              kind="layer", eps=0.1)
        return (q.double() * cq).sum() + (k.double() * ck).sum()
    for t in leaves:
        t.requires_grad_()
    grads = torch.autograd.grad(loss(leaves), leaves)
    along = sum((a.double() * d).sum() for a, d in zip(grads, dirs))
    h = 2.0 ** -7
    with torch.no_grad():
        diff = (loss([t + h * d for t, d in zip(leaves, dirs)]) - loss([t - h * d for t, d in zip(leaves, dirs)])) / (2 * h)
    size = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs))
    assert abs(float(along - diff)) <= 2e-4 * float(size)


def test_infinities_stay_in_their_row_and_pair(dev):
    """Without a norm an infinity reaches its pair alone, and features that are not turned
    keep their own; with one, its row."""
    rot = rotary_axes((16,), device=dev)
    x = torch.randn(1, 2, 6, 64, generator=torch.Generator().manual_seed(0)).to(BF)
    bad = x.clone()
    bad[0, 1, 2, 3], bad[0, 0, 4, 40] = math.inf, math.nan
    p = torch.arange(1, 7)[:, None].to(dev)
    y, z = rotate_heads(x.to(dev), p, rot).cpu(), rotate_heads(bad.to(dev), p, rot).cpu()
    same = torch.ones_like(x, dtype=torch.bool)
    same[0, 1, 2, 3] = same[0, 1, 2, 19] = same[0, 0, 4, 40] = False
    assert torch.equal(y[same], z[same]) and z[0, 0, 4, 40].isnan() and not z[0, 1, 2, 3].isfinite()
    a = qk_norm_rotate(bad.to(dev), x.to(dev), p, rot)[0].cpu()
    b = qk_norm_rotate(x.to(dev), x.to(dev), p, rot)[0].cpu()
    same[0, 1, 2] = same[0, 0, 4] = False
    assert torch.equal(a[same], b[same])


def test_empty_tensors(dev):
    rot = rotary_axes((8,), device=dev)
    w = torch.ones(16, device=dev, requires_grad=True)
    for shape in ((0, 2, 3, 16), (2, 2, 0, 16), (1, 0, 3, 16)):
        q = torch.zeros(shape, device=dev, requires_grad=True)
        p = torch.zeros(shape[2], 1, dtype=torch.int32, device=dev)
        oq, ok = qk_norm_rotate(q, q, p, rot, q_weight=w, k_weight=w)
        assert oq.shape == ok.shape == shape
        dw, = torch.autograd.grad(oq.sum() + ok.sum(), w)
        assert not dw.any()
    # heads of keys alone
    q, k = torch.zeros(2, 0, 3, 16, device=dev, requires_grad=True), torch.randn(2, 1, 3, 16, device=dev)
    oq, ok = qk_norm_rotate(q, k, torch.zeros(3, 1, dtype=torch.int32, device=dev), rot, q_weight=w, k_weight=w)
    assert oq.numel() == 0 and torch.isfinite(ok).all()
    dw, = torch.autograd.grad(oq.sum() + ok.sum(), w)
    assert dw.any()


def test_axes_outside_are_cut(dev):
    """A table's axis outside the positions reads the nearest one."""
    rot = rotary_axes((4, 4), device=dev)
    x, p = torch.randn(1, 1, 5, 16, device=dev), torch.arange(10, device=dev).view(5, 2)
    wild = rot._replace(axes=torch.tensor([-7] * 4 + [10 ** 9] * 4, dtype=torch.int32, device=dev))
    assert torch.equal(rotate_heads(x, p, rot), rotate_heads(x, p, wild))


def test_broadcast_and_overlapping_inputs(dev):
    """Heads that share memory, a gradient that is one number, rows that overlap."""
    rot = rotary_axes((16,), device=dev)
    p = torch.arange(6, device=dev)[:, None]
    one = torch.randn(2, 1, 6, 32, device=dev, requires_grad=True)
    y = rotate_heads(one.expand(2, 5, 6, 32), p, rot)
    assert torch.equal(y[:, 0], y[:, 4]) and torch.equal(y[:, :1], rotate_heads(one, p, rot))
    dx, = torch.autograd.grad(y.sum(), one)
    d1, = torch.autograd.grad(rotate_heads(one, p, rot).sum(), one)
    assert torch.allclose(dx, 5 * d1, atol=1e-5)
    slide = torch.randn(200, device=dev).unfold(0, 32, 8)[:6][None, None]
    assert torch.equal(rotate_heads(slide, p, rot), rotate_heads(slide.contiguous(), p, rot))


def test_captured_and_replayed(dev):
    """A decode step's call in a graph, replayed with new inputs; eager calls between."""
    rot = rotary_axes((64,), device=dev)
    q, k = torch.randn(8, 16, 1, 128, device=dev).to(BF), torch.randn(8, 4, 1, 128, device=dev).to(BF)
    w, p = torch.rand(128, device=dev).to(BF), torch.arange(8, device=dev).view(8, 1, 1)
    call = lambda: qk_norm_rotate(q, k, p, rot, q_weight=w, k_weight=w)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        q.normal_()
        p.add_(1000 * i)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_on_another_stream(dev):
    rot = rotary_axes((32,), device=dev)
    x, p = torch.randn(2, 3, 500, 64, device=dev), torch.arange(500, device=dev)[:, None]
    want = rotate_heads(x, p, rot)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate_heads(x, p, rot)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_the_aggregators_rotation(dev):
    """Blocks of 16 pairs with their own ladders and LayerNorm: `gpa::qk_norm_rope`'s tables
    say the same."""
    B, N, H = 1, 50, 4
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(B, N, 3 * H * 64, generator=g).to(BF).to(dev)
    par = [torch.randn(64, generator=g).to(dev) for _ in range(4)]
    grid = torch.stack((torch.arange(N) // 7, torch.arange(N) % 7), -1).int().to(dev)
    at = torch.arange(8)[:, None].double() * 100.0 ** (-torch.arange(16).double() / 16)
    table = torch.stack((at.cos(), at.sin()), -1).float().to(dev)
    want = _native.qk_norm_rope_params(qkv, par[0], par[1], par[2], par[3], 1e-5, grid, table, H, True, True)
    heads = qkv.view(B, N, 3, H, 64).permute(2, 0, 3, 1, 4)
    got = qk_norm_rotate(heads[0].float(), heads[1].float(), grid, rotary_axes((16, 16), base=100.0, ladder="own",
                         pairing="blocks", device=dev), q_weight=par[0], k_weight=par[1], q_bias=par[2], k_bias=par[3],
                         kind="layer", eps=1e-5)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=0, atol=64 * f * 12)


def test_registration(dev):
    """The dispatcher's checks of the op: schema, fake implementation, autograd."""
    rot = rotary_axes((3, 5), pairing="interleaved", device=dev)
    q, k = (torch.randn(2, h, 4, 20, device=dev, requires_grad=True) for h in (3, 1))
    w = torch.rand(20, device=dev, requires_grad=True)
    p = torch.arange(8, device=dev, dtype=torch.int32).view(4, 2)
    args = (q, k, p, rot.freqs, rot.axes, 1, [3, 5], w, w.detach(), None, None, 1, 1e-6)
    torch.library.opcheck(torch.ops.gpa.head_rotary.default, args)
    torch.library.opcheck(torch.ops.gpa.head_rotary.default, (q, None, p, rot.freqs, rot.axes, 1, [3, 5], None, None, None, None, 0, 0.0))


@pytest.mark.parametrize("dt,pdt", [(BF, BF), (BF, F), (F, F)])
@pytest.mark.parametrize("pairing", ["half", "interleaved"])
def test_parameters_at_any_address(dev, dt, pdt, pairing):
    """Parameters that begin between 16-byte pieces, beside heads that do not: the same bits."""
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, dq, dk = (torch.randn(2, h, 70, 64, generator=g, device=dev).to(dt) for h in (3, 2, 3, 2))
    flat = torch.randn(4 * 64 + 1, generator=g, device=dev).to(pdt)
    rotary, at = rotary_axes((32,), pairing=pairing), torch.arange(70, device=dev, dtype=torch.int32)[:, None]

    def run(par):
        leaves = [t.detach().requires_grad_() for t in (q, k, *par)]
        x, y, qw, kw, qb, kb = leaves
        out = qk_norm_rotate(x, y, at, rotary, q_weight=qw, k_weight=kw, q_bias=qb, k_bias=kb, kind="layer")
        return [*out, *torch.autograd.grad(out, leaves, [dq, dk])]
    views = [flat[1 + 64 * i:65 + 64 * i] for i in range(4)]
    assert views[0].data_ptr() % 16 and not q.data_ptr() % 16
    assert all(torch.equal(a, b) for a, b in zip(run(views), run([v.clone() for v in views])))

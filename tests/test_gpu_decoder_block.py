"""The language-model operators run together, as a decoder uses them: blocks of
`attention_masked` and `norm_gate_residual` in training, and decode steps with
`attention_shared_prefix` over a cache that grows, alone, captured and on two
streams.
"""
import math

import pytest
import torch
import torch.utils.checkpoint

from merging.fused_attention import attention_masked, attention_shared_prefix
from merging.fused_norms import norm_gate_residual
from oracle.masked_attention import masked_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


class _Plain(torch.autograd.Function):
    """The oracle's attention with its gradients, in 64 bits."""

    @staticmethod
    def forward(ctx, q, k, v, scale, kw):
        ctx.save_for_backward(q, k, v)
        ctx.args = scale, kw
        return masked_attention(q, k, v, scale, u=0.0, **kw).o

    @staticmethod
    def backward(ctx, d_o):
        q, k, v = ctx.saved_tensors
        scale, kw = ctx.args
        r = masked_attention(q, k, v, scale, u=0.0, d_o=d_o, **kw)
        return r.dq, r.dk, r.dv, None, None


def _blocks(x, layers, offsets, slopes, H, Hk, fused):
    """Two blocks of an attention-only decoder; x [B, S, C]."""
    B, S, C = x.shape
    D = C // H
    head = lambda t, n: t.view(B, S, n, D).transpose(1, 2)  # noqa: E731
    n = _rms(x, layers[0]["pre"])
    for i, w in enumerate(layers):
        q, k, v = (n @ w["qkv"]).split([H * D, Hk * D, Hk * D], -1)
        q, k, v = head(q, H), head(k, Hk), head(v, Hk)
        if fused:
            o = attention_masked(q, k, v, D ** -0.5, causal=True, cap=20.0, slopes=slopes, offsets=offsets).float()
        else:
            o = _Plain.apply(q, k, v, D ** -0.5, dict(causal=True, cap=20.0, slopes=slopes, offsets=offsets))
        y = o.transpose(1, 2).reshape(B, S, C) @ w["out"]
        after = layers[(i + 1) % len(layers)]["pre"]
        if fused:
            x, n = norm_gate_residual(x, y, after, post_weight=w["post"], gate=w["gate"], scale=0.5)
        else:
            x = x + 0.5 * w["gate"] * _rms(y, w["post"])
            n = _rms(x, after)
    return x, n


def test_training_blocks(dev):
    """fp32 activations, so the attention's 16-bit operands and results are all the
    rounding there is.  A gradient passes at most nine of them a block (q, k, v, P, o;
    dO, P, dS, and dq, dk or dv), of 2^-8 of a value at most, two blocks: 18 * 2^-8
    of the gradient's norm."""
    B, S, H, Hk, C = 2, 300, 4, 2, 256
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    layers = [dict(pre=1 + 0.1 * r(C), post=1 + 0.1 * r(C), gate=1 + 0.3 * r(C), qkv=r(C, 2 * C) / 16, out=r(C, C) / 16)
              for _ in range(2)]
    x, d_x, d_n = r(B, S, C), r(B, S, C), r(B, S, C)
    offsets, slopes = [[0, 17, 18, 300], [4, 100, 250, 290]], torch.tensor([0.5, 0.25, 0.1, 0.0])

    def grads(fused):
        cast = (lambda t: t.float().to(dev)) if fused else lambda t: t.clone()
        leaves = [cast(x)] + [cast(t) for w in layers for t in w.values()]
        for t in leaves:
            t.requires_grad_()
        it = iter(leaves[1:])
        ls = [{k: next(it) for k in w} for w in layers]
        off = torch.tensor(offsets, dtype=torch.int32, device=dev) if fused else offsets
        out = _blocks(leaves[0], ls, off, slopes.to(dev) if fused else slopes, H, Hk, fused)
        return [*out, *torch.autograd.grad(out, leaves, [cast(d_x), cast(d_n)])]
    got, want = grads(True), grads(False)
    names = ["x", "n", "dx"] + [f"{k}{i}" for i, w in enumerate(layers) for k in w]
    for name, a, b in zip(names, got, want):
        rel = ((a.detach().cpu().double() - b.detach()).norm() / b.norm()).item()
        assert rel <= 18 * 2.0 ** -8, (name, rel)


def _step(c, w):
    """A decode step's attention and the norms after it."""
    o = attention_shared_prefix(c["q"], c["pk"], c["pv"], c["k"], c["v"], 0.125, lengths=c["len"], cap=30.0)
    B, H, M, D = o.shape
    return (o, *norm_gate_residual(c["x"], o.transpose(1, 2).reshape(B, M, H * D), w, post_weight=w))


def _cache(dev, seed, B=5, H=6, Hk=2, P=700, N=90, D=64):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)  # noqa: E731
    return dict(q=r(B, H, 1, D), pk=r(Hk, P, D), pv=r(Hk, P, D), k=r(B, Hk, N, D), v=r(B, Hk, N, D),
                x=r(B, 1, H * D), len=torch.tensor([1, 90, 33, 64, 7][:B], dtype=torch.int32, device=dev))


def test_decode_steps(dev):
    """Each step's rows are those of one masked attention over the whole sequence.  Both
    round the weights and the output once: 2^-8 of sum p |v| and of |o| each."""
    c = _cache(dev, 1)
    c["len"] = torch.tensor([1, 60, 33, 64, 7], dtype=torch.int32, device=dev)
    w = torch.ones(384, device=dev, dtype=BF)
    B, P, N = 5, 700, 90
    for step in range(4):
        c["q"] = torch.randn_like(c["q"])
        at = c["len"].long()
        new = torch.randn(2, B, 2, 64, device=dev).to(BF)
        c["k"][torch.arange(B), :, at], c["v"][torch.arange(B), :, at] = new[0], new[1]
        c["len"] += 1
        o, h, n = _step(c, w)
        joined = [torch.cat((p.expand(B, -1, -1, -1), own), 2) for p, own in ((c["pk"], c["k"]), (c["pv"], c["v"]))]
        span = torch.stack((torch.zeros_like(c["len"]), P + c["len"]), 1)
        kw = dict(causal=True, cap=30.0, k_offsets=span)
        want = attention_masked(c["q"], *joined, 0.125, **kw)
        size = attention_masked(c["q"], joined[0], joined[1].abs(), 0.125, **kw).float() * (1 + 2 ** -6)
        assert ((o.float() - want.float()).abs() <= 2 * 2.0 ** -8 * (size + want.float().abs())).all()
        y = o.double().transpose(1, 2).reshape(B, 1, -1)
        ref = c["x"].double() + _rms(y, 1.0)
        assert ((h.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + 1e-5).all()
        assert ((n.double() - _rms(ref, 1.0)).abs() <= _rms(ref, 1.0).abs() * 2.0 ** -8 + 1e-5).all()
    assert N == c["k"].shape[2] and int(c["len"].max()) <= N


def test_decode_graphs_beside_eager_steps(dev):
    """Two captured steps, replayed on two streams at once and between eager ones, on
    contents and lengths that change."""
    w = (1 + 0.1 * torch.randn(384, device=dev)).to(BF)
    caches = [_cache(dev, 2), _cache(dev, 3, P=5000, N=2000)]
    graphs, outs = [], []
    for c in caches:
        _step(c, w)
    torch.cuda.synchronize()
    for c in caches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(c, w))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in caches]
    for turn in range(4):
        for c in caches:
            for name in ("q", "k", "v", "x"):
                c[name].copy_(torch.randn_like(c[name]))
            c["len"].copy_(torch.randint(1, c["k"].shape[2] + 1, (5,), device=dev))
        for graph, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for c, got in zip(caches, outs):
            for a, b in zip(got, _step(c, w)):
                assert torch.equal(a, b), turn


def test_training_on_two_streams(dev):
    """Two forward and backward passes of many row blocks at once give the bits that
    each gives alone."""
    g = torch.Generator(device=dev).manual_seed(5)
    r = lambda h: torch.randn(1, h, 2304, 64, generator=g, device=dev).to(BF)  # noqa: E731
    sets = [([r(8).requires_grad_(), r(8).requires_grad_(), r(8).requires_grad_()], r(8)) for _ in range(2)]
    off = torch.tensor([0, 700, 2304], dtype=torch.int32, device=dev)

    def step(x, d_o):
        o = attention_masked(*x, 0.125, causal=True, offsets=off)
        return [o.detach(), *torch.autograd.grad(o, x, d_o)]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, st in zip(sets, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([step(*s) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for runs, w in zip(got, want) for run in runs for a, b in zip(run, w))
    assert not math.isnan(float(want[0][0].float().sum()))


def test_compiled_and_checkpointed_blocks(dev):
    """A block traced as one graph, and one whose forward runs again in the backward
    pass, give the eager call's bits; a second derivative is refused."""
    g = torch.Generator(device=dev).manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF).requires_grad_()  # noqa: E731
    x, q, k, v = r(2, 130, 256), r(2, 4, 130, 64), r(2, 2, 130, 64), r(2, 2, 130, 64)
    w = torch.ones(256, device=dev, dtype=BF, requires_grad=True)
    off = torch.tensor([0, 40, 130], dtype=torch.int32, device=dev)

    def block(x, q, k, v, w):
        o = attention_masked(q, k, v, 0.125, causal=True, cap=20.0, offsets=off)
        return norm_gate_residual(x, o.transpose(1, 2).reshape(2, 130, 256), w, post_weight=w)
    leaves = [x, q, k, v, w]
    d = [torch.randn(2, 130, 256, generator=g, device=dev).to(BF) for _ in range(2)]

    def run(fn):
        out = fn(*leaves)
        return [*out, *torch.autograd.grad(out, leaves, d)]
    want = run(block)
    for fn in (torch.compile(block, backend="aot_eager", fullgraph=True),
               lambda *a: torch.utils.checkpoint.checkpoint(block, *a, use_reentrant=False)):
        assert all(torch.equal(a, b) for a, b in zip(run(fn), want))
    first = torch.autograd.grad(attention_masked(q, k, v, 0.125).float().square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().sum(), q)

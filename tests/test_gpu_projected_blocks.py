"""Whole decoder blocks of the framework's operators, as they are used together:
`linear_gate_residual` for the projections and the MLP, `qk_norm_rotate` by time, height
and width, and `attention_masked` in training or, in a step over drafted trees,
`draft_tree` and `attention_tree`.
"""
import math

import pytest
import torch
import torch.utils.checkpoint

from merging.fused_attention import attention_masked, attention_tree, draft_tree
from merging.fused_linear import linear_gate_residual
from merging.fused_rotary import qk_norm_rotate, rotary_axes

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
H, HK, D, C = 4, 2, 64, 256
SECTIONS = (8, 12, 12)


def _weights(seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    return dict(qkv=r(2 * C, C) / 16, q_w=1 + 0.2 * r(D), k_w=1 + 0.2 * r(D), out=r(C, H * D) / 16, g1=1 + 0.2 * r(C),
                up=r(3 * C, C) / 16, b_up=0.3 * r(3 * C), down=r(C, 3 * C) / 28, g2=0.5 + 0.2 * r(C))


def _heads(x, w):
    """q, k and v [B, heads, N, D], as they lie in the fused projection."""
    B, N, _ = x.shape
    y = linear_gate_residual(x, w["qkv"]).view(B, N, H + 2 * HK, D).transpose(1, 2)
    return y.split([H, HK, HK], 1)


def _rest(x, o, w):
    """The block's second half: both projections with gates and residuals."""
    B, N, _ = x.shape
    x = linear_gate_residual(o.transpose(1, 2).reshape(B, N, H * D), w["out"], gate=w["g1"], residual=x)
    h = linear_gate_residual(x, w["up"], w["b_up"], activation="gelu")
    return linear_gate_residual(h, w["down"], gate=w["g2"], residual=x)


def _block(x, places, offsets, w, rotary):
    q, k, v = _heads(x, w)
    q, k = qk_norm_rotate(q, k, places, rotary, q_weight=w["q_w"], k_weight=w["k_w"])
    return _rest(x, attention_masked(q, k, v, D ** -0.5, causal=True, offsets=offsets), w)


def _step(x, parents, lens, sizes, cache, w, rotary):
    """Drafted tokens x [B, T, C] behind their sequences' caches."""
    at, seen = draft_tree(parents, lens, sizes=sizes)
    q, k, v = _heads(x, w)
    q, k = qk_norm_rotate(q, k, at[..., None].expand(*at.shape, 3), rotary, q_weight=w["q_w"], k_weight=w["k_w"])
    return _rest(x, attention_tree(q, *cache, k, v, D ** -0.5, lengths=lens, seen=seen), w)


def _plain(x, places, mask, w, cache=None):
    """The block in 64 bits on the CPU; mask [B, N, keys], the cache's first."""
    B, N, _ = x.shape
    pairs = sum(SECTIONS)
    axis = torch.tensor([a for a, s in enumerate(SECTIONS) for _ in range(s)])
    t = places.double()[..., axis] * 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    cos, sin = (f(t).expand(B, N, pairs)[:, None] for f in (torch.cos, torch.sin))

    def turned(t, weight):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * weight
        a, b = t[..., :pairs], t[..., pairs:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    q, k, v = (x @ w["qkv"].t()).view(B, N, H + 2 * HK, D).transpose(1, 2).split([H, HK, HK], 1)
    q, k = turned(q, w["q_w"]), turned(k, w["k_w"])
    if cache is not None:
        k, v = torch.cat((cache[0], k), 2), torch.cat((cache[1], v), 2)
    k, v = (t.repeat_interleave(H // HK, 1) for t in (k, v))
    s = (q @ k.mT) * D ** -0.5
    s = s.masked_fill(~mask[:, None], -math.inf)
    some = mask.any(-1)[:, None, :, None]
    p = torch.where(some, torch.where(some, s, 0.0).softmax(-1), 0.0)
    x = x + w["g1"] * ((p @ v).transpose(1, 2).reshape(B, N, H * D) @ w["out"].t())
    z = x @ w["up"].t() + w["b_up"]
    return x + w["g2"] * ((0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)) @ w["down"].t())


def _places(N):
    """Frames of a 7 x 7 grid behind five special tokens."""
    at = torch.arange(N)
    cell = at % 54 - 5
    return torch.stack((at // 54, torch.where(cell < 0, 0, cell // 7 + 1), torch.where(cell < 0, 0, cell % 7 + 1)), -1).int()


def _near(name, got, want, roundings):
    rel = ((got.detach().cpu().double() - want.detach()).norm() / want.norm()).item()
    assert rel <= roundings * 2.0 ** -8, (name, rel)


def test_training_block(dev):
    """A gradient passes at most 21 roundings to bf16, of 2^-8 of the tensor's norm at most:
    forward the projection, q or k, P, o, x, the activation and the block's result; backward
    dz and the gradient of the input of four products (the residuals add into two of these, 2
    more), P, dS, dq, dk or dv, and the rotation's; and z, kept in fp16, an eighth of one."""
    B, N = 2, 130
    rotary = rotary_axes(SECTIONS)
    offsets = torch.tensor([[0, 17, 18, 130], [4, 60, 100, 128]], dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(B, N, C, generator=g).to(BF) for _ in range(2))
    at = torch.arange(N)
    mask = torch.zeros(B, N, N, dtype=torch.bool)
    for b, edges in enumerate(offsets.tolist()):
        for lo, hi in zip(edges, edges[1:]):
            own = (at >= lo) & (at < hi)
            mask[b] |= own[:, None] & own[None, :] & (at[None, :] <= at[:, None])

    def leaves(cast):
        w = {k: cast(t).requires_grad_() for k, t in _weights(1).items()}
        return cast(x).requires_grad_(), w
    xs, w = leaves(lambda t: t.to(dev))
    y = _block(xs, _places(N).to(dev), offsets.to(dev), w, rotary)
    got = [y, *torch.autograd.grad(y, [xs, *w.values()], dy.to(dev))]
    xs, w = leaves(lambda t: t.double())
    y = _plain(xs, _places(N), mask, w)
    want = [y, *torch.autograd.grad(y, [xs, *w.values()], dy.double())]
    for name, a, b in zip(["y", "dx", *("d_" + k for k in w)], got, want):
        _near(name, a, b, 7 if name == "y" else 21 + 0.125)


def _served(dev, seed, B, T, N):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).to(dev)  # noqa: E731
    ints = lambda *s, lo, hi: torch.randint(lo, hi, s, generator=g, dtype=torch.int32).to(dev)  # noqa: E731
    parents = torch.stack([ints(B, lo=-1, hi=max(i, 1)) for i in range(T)], 1)
    return dict(x=r(B, T, C), parents=parents, lens=ints(B, lo=0, hi=N + 1), sizes=ints(B, lo=0, hi=T + 1),
                cache=(r(B, HK, N, D), r(B, HK, N, D)))


@pytest.mark.parametrize("B,T,N", [(1, 1, 40), (3, 5, 700), (2, 40, 300), (5, 3, 0)])
def test_step_over_drafted_trees(dev, B, T, N):
    """The seven roundings of the forward; rows behind a sequence's size see nothing, and are what the
    block makes of no attention."""
    s, rotary = _served(dev, 10 + T, B, T, N), rotary_axes(SECTIONS)
    w = {k: t.to(dev) for k, t in _weights(2).items()}
    got = _step(s["x"], s["parents"], s["lens"], s["sizes"], s["cache"], w, rotary)
    places, mask = torch.zeros(B, T, 3, dtype=torch.int64), torch.zeros(B, T, N + T, dtype=torch.bool)
    for b in range(B):
        for i in range(int(s["sizes"][b])):
            chain = [i]
            while 0 <= int(s["parents"][b, chain[-1]]) < chain[-1]:
                chain.append(int(s["parents"][b, chain[-1]]))
            places[b, i] = int(s["lens"][b]) + len(chain) - 1
            mask[b, i, :int(s["lens"][b])] = True
            mask[b, i, [N + j for j in chain]] = True
    want = _plain(s["x"].cpu().double(), places, mask, {k: t.cpu().double() for k, t in w.items()},
                  [t.cpu().double() for t in s["cache"]])
    _near("y", got, want, 7)


def test_accepted_tokens_join_the_cache(dev):
    """A chain of drafted tokens, then the same tokens one step each over a cache that takes
    them up: the same rows, but for the order of sums.  Both round seven times."""
    B, N, T = 3, 200, 4
    s, rotary = _served(dev, 20, B, T, N), rotary_axes(SECTIONS)
    w = {k: t.to(dev) for k, t in _weights(4).items()}
    lens = torch.tensor([0, 77, 190], dtype=torch.int32, device=dev)
    chain = torch.arange(-1, T - 1, dtype=torch.int32, device=dev)
    want = _step(s["x"], chain, lens, None, s["cache"], w, rotary)
    ck, cv = (t.clone() for t in s["cache"])
    rows = torch.arange(B, device=dev)
    for i in range(T):
        x = s["x"][:, i:i + 1]
        y = _step(x, chain[:1], lens, None, (ck, cv), w, rotary)
        _near(f"token {i}", y, want[:, i:i + 1].cpu().double(), 14)
        _, k, v = _heads(x, w)
        _, k = qk_norm_rotate(k, k, lens[:, None, None].expand(B, 1, 3), rotary, q_weight=w["k_w"], k_weight=w["k_w"])
        ck[rows, :, lens.long()], cv[rows, :, lens.long()] = k[:, :, 0], v[:, :, 0]
        lens = lens + 1


def test_steps_in_graphs_on_two_streams(dev):
    """Two captured steps, replayed at once and between eager ones on trees, lengths and
    values that change, give the eager steps' bits."""
    rotary = rotary_axes(SECTIONS)
    w = {k: t.to(dev) for k, t in _weights(5).items()}
    sets = [_served(dev, 30, 3, 7, 900), _served(dev, 31, 2, 50, 3000)]
    run = lambda s: _step(s["x"], s["parents"], s["lens"], s["sizes"], s["cache"], w, rotary)  # noqa: E731
    for s in sets:
        run(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(s))
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(4):
        for s in sets:
            B, T, N = *s["parents"].shape, s["cache"][0].shape[2]
            new = _served(dev, 40 + turn, B, T, N)
            for name in ("x", "parents", "lens", "sizes"):
                s[name].copy_(new[name])
            for a, b in zip(s["cache"], new["cache"]):
                a.copy_(b)
        for graph, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for s, got in zip(sets, outs):
            assert torch.equal(got, run(s)), turn


def test_training_on_two_streams_compiled_and_checkpointed(dev):
    """Forward and backward of a block on two streams at once, traced as one graph, and with
    its forward run again in the backward, give the bits that an eager call gives alone."""
    rotary = rotary_axes(SECTIONS)
    offsets, places = torch.tensor([0, 40, 600], dtype=torch.int32, device=dev), _places(600).to(dev)
    g = torch.Generator(device=dev).manual_seed(9)
    sets = [(torch.randn(1, 600, C, generator=g, device=dev).to(BF).requires_grad_(),
             {k: t.to(dev).requires_grad_() for k, t in _weights(6 + i).items()}) for i in range(2)]
    dy = torch.randn(1, 600, C, generator=g, device=dev).to(BF)

    def block(x, *w):
        return _block(x, places, offsets, dict(zip(sets[0][1], w)), rotary)

    def run(s, fn=block):
        leaves = [s[0], *s[1].values()]
        y = fn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for s, st in zip(sets, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([run(s) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for runs, one in zip(got, want) for r in runs for a, b in zip(r, one))
    for fn in (torch.compile(block, backend="aot_eager", fullgraph=True),
               lambda *a: torch.utils.checkpoint.checkpoint(block, *a, use_reentrant=False)):
        assert all(torch.equal(a, b) for a, b in zip(run(sets[0], fn), want[0]))

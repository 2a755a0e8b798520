"""`draft_tree` and `attention_tree` against the 64-bit definition: a drafted token is
the last query of a sequence of its own, the cache's keys, its ancestors and itself.
Tolerances: the oracle's elementwise bounds (one rounding of each weight and
result; the join is fp32)."""
import math
import random

import pytest
import torch

from merging import _native
from merging.fused_attention import attention_masked, attention_tree, draft_tree
from oracle.masked_attention import masked_attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _chain(parents, i):
    """The ancestors of token i and itself, first to last."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out[::-1]


def _trees(kind, B, T, seed):
    rng = random.Random(seed)
    if kind == "chain":
        return [[i - 1 for i in range(T)] for _ in range(B)]
    if kind == "roots":
        return [[-1] * T for _ in range(B)]
    if kind == "wild":                                       # none an earlier token's number but by chance
        return [[rng.choice([-9, i, i + 1, 2 ** 31 - 1, -2 ** 31, rng.randint(-1, T)]) for i in range(T)] for _ in range(B)]
    return [[rng.randint(max(-1, i - 6), i - 1) for i in range(T)] for _ in range(B)]


def _check(dev, B, H, Hk, T, N, lens, D=64, dt=BF, kind="random", sizes=None, cap=None, slopes=None, seed=0,
           layout="bhnd", bad=True, rows=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, ck, cv, k, v = (t.to(dt) for t in (r(B, H, T, D) * 1.3, r(B, Hk, N, D) * 1.3, r(B, Hk, N, D),
                                          r(B, Hk, T, D) * 1.3, r(B, Hk, T, D)))
    parents = _trees(kind, B, T, seed)
    there = sizes or [T] * B
    if bad:                                                  # what a row does not see is anything
        for b in range(B):
            n = min(max(lens[b], 0), N)
            ck[b, :, n:], cv[b, :, n:] = math.nan, math.inf
            k[b, :, max(there[b], 0):], v[b, :, max(there[b], 0):] = math.inf, math.nan
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ln, sz = ints(lens), None if sizes is None else ints(sizes)
    at, seen = draft_tree(ints(parents), ln, sizes=sz)
    on = [t.to(dev) for t in (q, ck, cv, k, v)]
    if layout == "bnhd":                                     # as projections and caches by token lay them out
        on = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in on]
    if layout == "odd":
        on = [torch.nn.functional.pad(t, (3, 2))[..., 3:-2] for t in on]
    sl = None if slopes is None else slopes.to(dev)
    call = lambda: attention_tree(*on, D ** -0.5, lengths=ln, seen=seen, cap=cap, slopes=sl, return_lse=True)  # noqa: E731
    o, lse = call()
    assert o.shape == q.shape and o.dtype == dt and lse.shape == q.shape[:3]
    slack = 2.0 ** -24 if dt == HF else 0.0
    rng = random.Random(seed)
    for b in range(B):
        size, n = min(max(there[b], 0), T), min(max(lens[b], 0), N)
        got_bits = [[j for j in range(T) if seen[b, i, j // 32].item() >> (j % 32) & 1] for i in range(T)] \
            if T <= 70 else None
        for i in range(T):
            if i >= size:
                assert at[b, i] == 0 and not seen[b, i].any()
                assert not o[b, :, i].any() and (lse[b, :, i] == -math.inf).all()
                continue
            chain = _chain(parents[b], i)
            assert at[b, i] == lens[b] + len(chain) - 1
            assert got_bits is None or got_bits[i] == chain
            if rows is not None and rng.random() > rows:
                continue
            keys = torch.cat((ck[b, :, :n], k[b][:, chain]), 1)[None]
            values = torch.cat((cv[b, :, :n], v[b][:, chain]), 1)[None]
            ref = masked_attention(q[b:b + 1, :, i:i + 1], keys, values, D ** -0.5, cap=cap, slopes=slopes, causal=True,
                                   offsets=[0, 1], k_offsets=[0, keys.shape[2]], u=torch.finfo(dt).eps / 2)
            off = (o[b, :, i].cpu().double() - ref.o[0, :, 0]).abs()
            assert (off <= ref.o_bound[0, :, 0] + slack).all(), (b, i, float((off / ref.o_bound[0, :, 0]).max()))
            assert ((lse[b, :, i].cpu().double() - ref.lse[0, :, 0]).abs() <= ref.lse_bound).all()
    again = call()
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Hk,T,N,lens,sizes", [
    (1, 1, 1, 1, 1, [1], None),
    (1, 2, 2, 1, 0, [0], None),                              # no cache at all
    (2, 4, 2, 7, 100, [100, 33], [7, 3]),
    (3, 6, 2, 5, 40, [0, 1, 40], [5, 0, 1]),                 # an empty cache, a sequence without a draft
    (2, 8, 1, 33, 70, [64, 65], [33, 32]),                   # more than 128 rows; words that end inside
    (2, 4, 4, 40, 1500, [1500, 700], None),
    (4, 16, 4, 8, 3000, [2999, 31, 32, 1024], [8, 8, 1, 7]),
    (5, 4, 2, 64, 300, [299, 1, 0, 300, 128], [64, 63, 1, 33, 64]),
])
def test_against_64_bits(dev, dt, D, B, H, Hk, T, N, lens, sizes):
    _check(dev, B, H, Hk, T, N, lens, D=D, dt=dt, sizes=sizes)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("kw", [
    dict(kind="chain"), dict(kind="roots"), dict(kind="wild"), dict(cap=7.0), dict(cap=50.0, D=128), dict(slopes="up"),
    dict(slopes="down"), dict(slopes="up", cap=20.0, dt=HF, D=128), dict(slopes="down", dt=HF), dict(layout="bnhd"),
    dict(layout="odd"), dict(lens=[-5, 10 ** 9]), dict(sizes=[-1, 99]), dict(bad=False), dict(seed=4, kind="wild", slopes="up")])
def test_options(dev, few, kw):
    H, T = (4, 6) if few else (8, 37)
    kw = dict(kw)
    if "slopes" in kw:
        sign = 1 if kw["slopes"] == "up" else -0.05
        kw["slopes"] = torch.tensor([sign * 2.0 ** -(i + 1) for i in range(H)])
    _check(dev, 2, H, 2, T, 600, kw.pop("lens", [577, 130]), **kw)


@pytest.mark.parametrize("B,H,Hk,T,N", [(70, 2, 1, 3, 90), (130, 1, 1, 2, 400), (3, 2, 1, 200, 100), (1, 2, 1, 1024, 40),
                                        (1, 2, 2, 16, 20_001), (2, 8, 2, 64, 9000), (1, 1, 1, 1, 70_000), (20, 16, 4, 16, 2500)])
@pytest.mark.parametrize("dt", [BF, HF])
def test_sizes(dev, dt, B, H, Hk, T, N):
    """Many sequences, long drafts and caches, pieces of unequal sequences."""
    rng = random.Random(B * N)
    lens = [N - (i * 7919) % N if i % 3 else rng.randint(0, N) for i in range(B)]
    _check(dev, B, H, Hk, T, N, lens, dt=dt, rows=min(1.0, 60 / (B * T)), sizes=[rng.randint(0, T) for _ in range(B)])


def test_a_chain_is_causal_attention(dev):
    """A draft in a line over a cache: the same as causal attention over both."""
    g = torch.Generator().manual_seed(1)
    B, H, Hk, T, N, D = 2, 8, 2, 12, 500, 128
    r = lambda *s: torch.randn(*s, generator=g).to(BF).to(dev)  # noqa: E731
    q, ck, cv, k, v = r(B, H, T, D), r(B, Hk, N, D), r(B, Hk, N, D), r(B, Hk, T, D), r(B, Hk, T, D)
    parents = torch.arange(-1, T - 1, dtype=torch.int32, device=dev)
    at, seen = draft_tree(parents, torch.full((B,), N, dtype=torch.int32, device=dev))
    assert torch.equal(at, torch.arange(N, N + T, device=dev).int().expand(B, T))
    o, lse = attention_tree(q, ck, cv, k, v, 0.1, seen=seen, return_lse=True)
    want, wlse = attention_masked(q, torch.cat((ck, k), 2), torch.cat((cv, v), 2), 0.1, causal=True, offsets=torch.tensor(
        [0, T], dtype=torch.int32, device=dev), k_offsets=torch.tensor([0, N + T], dtype=torch.int32, device=dev), return_lse=True)
    # two roundings of outputs of norm 1 and of weights that add to one
    assert (o.float() - want.float()).abs().max() <= 4 * 2.0 ** -8 * want.float().abs().max()
    assert (lse - wlse).abs().max() <= 2e-5


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [5, 40])
def test_infinities_reach_the_rows_that_see_them(dev, D, T):
    """A sibling's infinite values stay with it and its descendants; large finite values
    (bf16) keep finite outputs."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    q, ck, cv, k, v = r(1, 2, T, D), r(1, 1, 64, D), r(1, 1, 64, D), r(1, 1, T, D), r(1, 1, T, D)
    parents = [-1, -1] + [i % 2 for i in range(T - 2)]      # two roots, the others hang on one of them
    ln = torch.tensor([50], dtype=torch.int32, device=dev)
    _, seen = draft_tree(torch.tensor(parents, dtype=torch.int32, device=dev), ln)
    run = lambda v: attention_tree(q.to(dev), ck.to(dev), cv.to(dev), k.to(dev), v.to(dev), 0.2, lengths=ln, seen=seen).cpu()  # noqa: E731
    w = v.clone()
    w[0, 0, 1, 3], w[0, 0, 1, 4], w[0, 0, 1, 5] = math.inf, -math.inf, math.nan
    a, b = run(v), run(w)
    hit = torch.tensor([1 in _chain(parents, i) for i in range(T)])
    # rows that do not see it: the same but for the order of the careful walk's roundings
    assert (a[:, :, ~hit].float() - b[:, :, ~hit].float()).abs().max() <= 3 * 2.0 ** -8
    assert (b[0, :, hit, 3] == math.inf).all() and (b[0, :, hit, 4] == -math.inf).all() and b[0, :, hit, 5].isnan().all()
    assert torch.isfinite(b[0, :, hit, 6:]).all()
    big = run(torch.full_like(v, 3e38))
    assert torch.isfinite(big).all()
    q2 = torch.full_like(q, 30.0)
    far = attention_tree(q2.to(dev), ck.to(dev), cv.to(dev) * 3e37, torch.full_like(k, 3.0).to(dev), v.to(dev) * 1e37, 0.2,
                         lengths=ln, seen=seen)
    assert torch.isfinite(far).all()


def test_bits_of_other_making(dev):
    """Rows of bits that are no tree's: a token may see any drafted ones; bits behind the last
    token count for nothing."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    T, N, D = 20, 70, 64
    q, ck, cv, k, v = r(1, 1, T, D), r(1, 1, N, D), r(1, 1, N, D), r(1, 1, T, D), r(1, 1, T, D)
    see = torch.rand(T, T, generator=g) < 0.4
    see[3] = False
    words = [sum(1 << j for j in range(T) if see[i, j]) | (0xfff << 20) for i in range(T)]
    seen = torch.tensor([w - (1 << 32) if w >> 31 else w for w in words], dtype=torch.int32, device=dev).view(1, T, 1)
    o = attention_tree(*(t.to(dev) for t in (q, ck, cv, k, v)), 0.3, seen=seen).cpu()
    for i in range(T):
        if not see[i].any():
            assert not o[0, 0, i].any()
            continue
        keys, values = torch.cat((ck[0, 0], k[0, 0, see[i]])).double(), torch.cat((cv[0, 0], v[0, 0, see[i]])).double()
        w = torch.softmax(keys @ q[0, 0, i].double() * 0.3, 0)
        want, size = w @ values, w @ values.abs()
        assert ((o[0, 0, i].double() - want).abs() <= 2.0 ** -8 * (want.abs() + 2.2 * size) + 1e-5).all()


def test_captured_and_replayed(dev):
    """A step's calls in a graph, whose lengths, trees and keys change between replays; two
    graphs at once have workspaces of their own."""
    B, H, Hk, T, N, D = 3, 8, 2, 16, 4000, 64
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).to(dev)  # noqa: E731
    q, ck, cv, k, v = r(B, H, T, D), r(B, Hk, N, D), r(B, Hk, N, D), r(B, Hk, T, D), r(B, Hk, T, D)
    ln = torch.tensor([4000, 17, 900], dtype=torch.int32, device=dev)
    parents = torch.tensor(_trees("random", B, T, 0), dtype=torch.int32, device=dev)

    def step():
        at, seen = draft_tree(parents, ln)
        return at, attention_tree(q, ck, cv, k, v, 0.125, lengths=ln, seen=seen)
    step()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for i in range(4):
        ln.copy_(torch.tensor([[4000, 17, 900], [0, 4000, 3999], [5, 5, 5], [2000, 2100, 2200]][i], dtype=torch.int32))
        parents.copy_(torch.tensor(_trees("random", B, T, i + 1), dtype=torch.int32))
        q.normal_(generator=None)
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in outs:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_on_another_stream(dev):
    B, H, Hk, T, N, D = 2, 4, 2, 9, 3000, 64
    r = lambda *s: torch.randn(*s, device=dev).to(HF)  # noqa: E731
    q, ck, cv, k, v = r(B, H, T, D), r(B, Hk, N, D), r(B, Hk, N, D), r(B, Hk, T, D), r(B, Hk, T, D)
    ln, par = torch.tensor([2000, 3000], dtype=torch.int32, device=dev), torch.full((T,), -1, dtype=torch.int32, device=dev)

    def step():
        _, seen = draft_tree(par, ln)
        return attention_tree(q, ck, cv, k, v, 0.125, lengths=ln, seen=seen)
    want, side = step(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        here = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(here, want)


def test_empty(dev):
    z = lambda *s: torch.zeros(*s, dtype=BF, device=dev)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    at, seen = draft_tree(i(0, 4), i(0))
    assert at.shape == (0, 4) and seen.shape == (0, 4, 1)
    at, seen = draft_tree(i(2, 0), i(2))
    assert at.shape == (2, 0) and seen.shape == (2, 0, 0)
    assert attention_tree(z(2, 4, 0, 64), z(2, 2, 9, 64), z(2, 2, 9, 64), z(2, 2, 0, 64), z(2, 2, 0, 64), 1.0, seen=seen).numel() == 0
    assert attention_tree(z(0, 4, 3, 64), z(0, 2, 9, 64), z(0, 2, 9, 64), z(0, 2, 3, 64), z(0, 2, 3, 64), 1.0,
                          seen=i(0, 3, 1)).numel() == 0


def test_registration(dev):
    r = lambda *s: torch.randn(*s, device=dev).to(BF)  # noqa: E731
    par, ln = torch.tensor([-1, 0, 0], dtype=torch.int32, device=dev), torch.tensor([9, 4], dtype=torch.int32, device=dev)
    torch.library.opcheck(torch.ops.gpa.draft_tree.default, (par, ln, None))
    _, seen = draft_tree(par, ln)
    torch.library.opcheck(torch.ops.gpa.attn_tree.default, (
        r(2, 4, 3, 64), r(2, 2, 9, 64), r(2, 2, 9, 64), r(2, 2, 3, 64), r(2, 2, 3, 64), ln, seen, 0.125, 0.0, None, True))
    q = r(2, 4, 3, 64).requires_grad_()
    out = attention_tree(q, r(2, 2, 9, 64), r(2, 2, 9, 64), r(2, 2, 3, 64), r(2, 2, 3, 64), 0.125, lengths=ln, seen=seen)
    with pytest.raises(RuntimeError, match="forward-only"):
        out.sum().backward()
    assert _native.MAX_DRAFT == 1024

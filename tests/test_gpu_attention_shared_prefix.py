"""`attention_shared_prefix` against the 64-bit definition (each sequence's
prefix and own keys as one causal document), and against `attention_masked`
over the joined keys.  Tolerances: the oracle's elementwise bounds (one
rounding of each weight and result; the join is fp32)."""
import math

import pytest
import torch

from merging.fused_attention import attention_masked, attention_shared_prefix
from oracle.masked_attention import masked_attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _inputs(B, H, Hk, M, P, N, D, dt, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [t.to(dt) for t in (r(B, H, M, D) * 1.3, r(Hk, P, D) * 1.3, r(Hk, P, D), r(B, Hk, N, D) * 1.3,
                               r(B, Hk, N, D))]


def _check(dev, B, H, Hk, M, P, N, D, dt, lens, cap=None, slopes=None, seed=0):
    q, pk, pv, k, v = _inputs(B, H, Hk, M, P, N, D, dt, seed)
    for b, n in enumerate(lens):                             # what lies behind a sequence is anything
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.inf
    on = [t.to(dev) for t in (q, pk, pv, k, v)]
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    sl = None if slopes is None else slopes.to(dev)
    o, lse = attention_shared_prefix(*on, D ** -0.5, lengths=ln, cap=cap, slopes=sl, return_lse=True)
    assert o.shape == q.shape and o.dtype == dt and lse.shape == q.shape[:3]
    slack = 2.0 ** -24 if dt == HF else 0.0
    for b, n in enumerate(lens):
        keys = torch.cat((pk, k[b, :, :n]), 1)[None]
        values = torch.cat((pv, v[b, :, :n]), 1)[None]
        # the queries are the last M own tokens, whether or not that many are there
        off = dict(offsets=[0, M], k_offsets=[0, P + n])
        ref = masked_attention(q[b:b + 1], keys, values, D ** -0.5, cap=cap, slopes=slopes, causal=True,
                               prefix=P, u=torch.finfo(dt).eps / 2, **off)
        got, bound = o[b].cpu().double(), ref.o_bound[0] + slack
        bad = ~((got - ref.o[0]).abs() <= bound)
        assert not bad.any(), (b, n, int(bad.sum()), got[bad][:4], ref.o[0][bad][:4])
        want = ref.lse[0]
        empty = want == -math.inf
        assert torch.equal(lse[b].cpu() == -math.inf, empty)
        assert ((lse[b].cpu().double() - want)[~empty].abs() <= ref.lse_bound).all()
    assert torch.equal(attention_shared_prefix(*on, D ** -0.5, lengths=ln, cap=cap, slopes=sl), o)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Hk,M,P,lens", [
    (1, 1, 1, 1, 1, [1]),
    (3, 4, 2, 1, 500, [1, 64, 33]),
    (4, 6, 2, 3, 33, [3, 0, 2, 70]),          # an empty sequence, one shorter than its queries
    (9, 8, 1, 1, 1025, [5] * 9),
    (2, 2, 2, 130, 200, [130, 150]),           # a whole chunk of new tokens
    (2, 14, 2, 2, 31, [2, 9]),
])
def test_against_the_definition(dev, B, H, Hk, M, P, lens, D, dt):
    _check(dev, B, H, Hk, M, P, max(lens) + 5, D, dt, lens, seed=P)
    _check(dev, B, H, Hk, M, P, max(max(lens), 1), D, dt, lens, cap=20.0, slopes=torch.rand(H) * 0.2, seed=P + 1)


def test_long_prefix(dev):
    _check(dev, 5, 8, 2, 1, 20_011, 300, 64, BF, [300, 1, 77, 250, 31], slopes=torch.full((8,), 0.01))
    _check(dev, 40, 8, 2, 2, 5000, 700, 128, HF, [700 - 17 * i for i in range(40)], cap=30.0)


def test_no_prefix_and_no_own_keys(dev):
    q, pk, pv, k, v = (t.to(dev) for t in _inputs(2, 4, 2, 3, 50, 40, 64, BF, 1))
    want = attention_masked(q, k, v, 0.125, causal=True)
    assert torch.equal(attention_shared_prefix(q, pk[:, :0], pv[:, :0], k, v, 0.125), want)
    want = attention_masked(q, pk.expand(2, 2, 50, 64), pv.expand(2, 2, 50, 64), 0.125).float()
    got = attention_shared_prefix(q, pk, pv, k[:, :, :0], v[:, :, :0], 0.125).float()
    # both round the same weights to bf16, and their own results: two half steps and a
    # last bit of the fp32 join
    assert ((got - want).abs() <= 2 * 2.0 ** -8 * want.abs() + 1e-6).all()
    assert attention_shared_prefix(q[:0], pk, pv, k[:0], v[:0], 0.125).shape == (0, 4, 3, 64)


def test_strides_and_graph(dev):
    """Caches as rows of several heads, a prefix inside a longer buffer, lengths
    that grow between the replays of a graph."""
    B, H, Hk, D, P = 3, 4, 2, 64, 90
    g = torch.Generator(device=dev).manual_seed(0)
    rows = torch.randn(B, 64, 2 * Hk, D, generator=g, device=dev).to(BF)
    buf = torch.randn(P + 20, 2 * Hk, D, generator=g, device=dev).to(BF)
    k, v = rows[:, :, :Hk].transpose(1, 2), rows[:, :, Hk:].transpose(1, 2)
    pk, pv = buf[:P, :Hk].transpose(0, 1), buf[:P, Hk:].transpose(0, 1)
    q = torch.randn(B, 1, H, D, generator=g, device=dev).to(BF).transpose(1, 2)
    lens = torch.tensor([1, 20, 64], dtype=torch.int32, device=dev)
    plain = lambda: attention_shared_prefix(q.contiguous(), pk.contiguous(), pv.contiguous(),  # noqa: E731
                                            k.contiguous(), v.contiguous(), 0.125, lengths=lens)
    call = lambda: attention_shared_prefix(q, pk, pv, k, v, 0.125, lengths=lens)  # noqa: E731
    assert torch.equal(call(), plain())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for step in range(4):
        lens.copy_(torch.tensor([1 + step, 20 + 3 * step, 64 - step], dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g, device=dev))
        want = plain()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want), step


def test_lengths_outside_the_cache_are_cut(dev):
    q, pk, pv, k, v = (t.to(dev) for t in _inputs(3, 2, 2, 1, 10, 40, 64, BF, 1))
    lens = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = attention_shared_prefix(q, pk, pv, k, v, 0.125, lengths=lens(-5, 1000, 2 ** 31 - 1))
    want = attention_shared_prefix(q, pk, pv, k, v, 0.125, lengths=lens(0, 40, 40))
    assert torch.equal(got, want)


def test_op_check(dev):
    q, pk, pv, k, v = (t.to(dev) for t in _inputs(2, 4, 2, 3, 50, 40, 64, BF, 1))
    torch.library.opcheck(torch.ops.gpa.attn_shared_prefix.default,
                          (q, pk, pv, k, v, None, 0.125, 0.0, None, True))

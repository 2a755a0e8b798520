"""`attention_masked` and its gradients against the 64-bit definition
(oracle/masked_attention.py): documents, causal and prefix masks, caps,
slopes, shared heads, padded batches, strides, rows that see nothing, values
that no row may see.

Every tolerance is the oracle's elementwise bound: one rounding (half a step)
of each weight and of each result in the operands' format, fp32 scores and
sums.  fp16 results below 2^-14 are rounded to steps of 2^-24, which is added.
"""
import math

import pytest
import torch

from merging.fused_attention import attention_masked
from oracle.masked_attention import masked_attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _inputs(B, H, Hk, M, N, D, dt, seed, std=1.3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = r(B, H, M, D) * std, r(B, Hk, N, D) * std, r(B, Hk, N, D)
    return [t.to(dt) for t in (q, k, v, r(B, H, M, D))] + [r(B, H, M) * 0.1]


def _near(name, got, want, bound, dt):
    got = got.detach().cpu().double()
    slack = 2.0 ** -24 if dt == HF else 0.0
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound + slack)
    assert not bad.any(), (name, int(bad.sum()), got[bad][:4], want[bad][:4], bound[bad][:4])


def _check(dev, B, H, Hk, M, N, D, dt, seed=0, back=True, with_lse_grad=False, slopes=None, prefix=None,
           offsets=None, k_offsets=None, **kw):
    q, k, v, d_o, d_lse = _inputs(B, H, Hk, M, N, D, dt, seed)
    scale = D ** -0.5
    ref = masked_attention(q, k, v, scale, slopes=slopes, prefix=0 if prefix is None else prefix,
                           offsets=offsets, k_offsets=k_offsets, d_o=d_o if back else None,
                           d_lse=d_lse if with_lse_grad else None, u=torch.finfo(dt).eps / 2, **kw)
    on = lambda t: None if t is None else torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    if isinstance(prefix, list):
        prefix = on(prefix)
    args = dict(slopes=None if slopes is None else slopes.to(dev), prefix=prefix, offsets=on(offsets),
                k_offsets=on(k_offsets), **kw)
    q, k, v, d_o, d_lse = (t.to(dev) for t in (q, k, v, d_o, d_lse))
    o, lse = attention_masked(q, k, v, scale, return_lse=True, **args)
    _near("o", o, ref.o, ref.o_bound, dt)
    empty = ref.lse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    assert ((lse.cpu().double() - ref.lse)[~empty].abs() <= ref.lse_bound).all()
    assert torch.equal(attention_masked(q, k, v, scale, **args), o)
    if not back:
        return
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o2, lse2 = attention_masked(q, k, v, scale, return_lse=True, **args)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    lse2 = torch.where(torch.isinf(lse2), torch.zeros_like(lse2), lse2)
    outs, gouts = ([o2, lse2], [d_o, d_lse]) if with_lse_grad else ([o2], [d_o])
    grads = torch.autograd.grad(outs, leaves, gouts)
    for name, got, want, bound in zip("qkv", grads, (ref.dq, ref.dk, ref.dv),
                                      (ref.dq_bound, ref.dk_bound, ref.dv_bound)):
        assert got.dtype == dt
        _near("d" + name, got, want, bound, dt)
    o3 = attention_masked(q, k, v, scale, **args)
    again = torch.autograd.grad([o3], leaves, [d_o]) if not with_lse_grad else grads
    assert all(torch.equal(a, b) for a, b in zip(grads, again))          # no order changes a bit


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 33), (31, 32), (33, 31), (128, 128), (129, 257), (300, 5)])
def test_one_document(dev, M, N, D, dt):
    _check(dev, 2, 2, 2, M, N, D, dt, seed=M + N)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(4, 1), (6, 2), (5, 1), (32, 1), (40, 1)])
def test_causal_with_shared_heads(dev, heads, D, dt):
    _check(dev, 1, *heads, 77, 77, D, dt, seed=heads[0], causal=True)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("cap", [None, 5.0, 50.0])
@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_scores(dev, D, slope, cap, dt):
    slopes = torch.tensor([0.5, 0.0, 0.03, 2.0]) if slope else None
    _check(dev, 2, 4, 2, 150, 150, D, dt, seed=3, causal=True, cap=cap, slopes=slopes, with_lse_grad=True)
    if slope:
        _check(dev, 2, 4, 2, 40, 90, D, dt, seed=4, cap=cap, slopes=torch.rand(2, 4), prefix=7, causal=True)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("causal,prefix", [(False, None), (True, None), (True, 4), (True, [0, 9, 500, 1, 3])])
@pytest.mark.parametrize("offsets", [
    [0, 40, 41, 41, 170, 200],                    # a document of one token, one of none
    [0, 0, 128, 129, 160, 200],
    [7, 30, 62, 64, 150, 190],                    # tokens of no document at both ends
    [[0, 10, 20, 30, 40, 200], [5, 100, 100, 100, 100, 100]],
])
def test_documents(dev, offsets, causal, prefix, dt):
    _check(dev, 2, 4, 2, 200, 200, 64, dt, seed=11, causal=causal, prefix=prefix, offsets=offsets)
    _check(dev, 2, 3, 3, 200, 200, 128, dt, seed=12, causal=causal, prefix=prefix, offsets=offsets, cap=20.0)


@pytest.mark.parametrize("causal", [False, True])
def test_documents_of_other_key_lengths(dev, causal):
    """More keys than queries (a cache), fewer (queries that see nothing), none."""
    off, koff = [0, 5, 40, 60, 61], [0, 70, 80, 80, 200]
    _check(dev, 1, 4, 2, 64, 230, 64, BF, seed=5, causal=causal, offsets=off, k_offsets=koff,
           slopes=torch.tensor([1.0, 0.1, 0.2, 0.5]))
    _check(dev, 1, 2, 2, 64, 230, 128, HF, seed=6, causal=causal, offsets=off, k_offsets=koff,
           prefix=3 if causal else None)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M", [1, 3])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (64, 7)])
def test_padded_batch_of_new_tokens(dev, D, G, M, dt):
    """A decode step: ragged cache lengths, one of them 0, keys split over workgroups."""
    lens = [[0, n] for n in (3000, 1, 0, 2047, 700)]
    _check(dev, 5, 2 * G, 2, M, 3000, D, dt, seed=M, back=False, causal=True, k_offsets=lens, cap=30.0)
    _check(dev, 5, 2 * G, 2, M, 3000, D, dt, seed=M + 9, causal=True, k_offsets=lens)


def test_long_and_wide(dev):
    _check(dev, 1, 2, 1, 1500, 1500, 128, BF, seed=1, causal=True, cap=50.0)
    _check(dev, 1, 1, 1, 1333, 2100, 64, HF, seed=2)
    _check(dev, 1, 1, 1, 2, 40_000, 64, BF, seed=3, back=False, causal=True, slopes=torch.tensor([0.01]))


def test_blocks_of_unequal_length(dev):
    """Many row blocks under a mask: cut and taken in order of their lengths."""
    _check(dev, 1, 8, 8, 2100, 2100, 64, BF, seed=21, back=False, causal=True, slopes=torch.rand(8))
    _check(dev, 1, 8, 8, 2100, 2100, 128, HF, seed=22, back=False, causal=True, prefix=900, cap=20.0)
    off = [40, 41, 600, 600, 1990, 2060]
    _check(dev, 1, 12, 4, 2100, 2100, 128, BF, seed=23, back=False, offsets=off)
    _check(dev, 1, 15, 5, 2100, 2100, 64, HF, seed=24, back=False, offsets=off, causal=True, prefix=[1, 0, 5, 3000, 2])
    lens = [[0, n] for n in (2100, 0, 1, 2099, 64, 1025)]
    _check(dev, 6, 22, 11, 70, 2100, 64, BF, seed=25, back=False, causal=True, k_offsets=lens, cap=30.0)
    _check(dev, 6, 22, 11, 70, 2100, 128, BF, seed=26, back=False, k_offsets=lens)


def test_gradients_of_blocks_of_unequal_length(dev):
    _check(dev, 1, 8, 8, 2100, 2100, 64, BF, seed=31, causal=True, slopes=torch.rand(8))
    _check(dev, 1, 8, 8, 2100, 2100, 128, HF, seed=32, causal=True, prefix=900, cap=20.0)
    off = [40, 41, 600, 600, 1990, 2060]
    _check(dev, 1, 12, 4, 2100, 2100, 128, BF, seed=33, offsets=off, with_lse_grad=True)
    _check(dev, 1, 15, 5, 2100, 2100, 64, HF, seed=34, offsets=off, causal=True, prefix=[1, 0, 5, 3000, 2])
    lens = [[0, n] for n in (2100, 0, 1, 2099, 64, 1025)]
    _check(dev, 6, 33, 3, 190, 2100, 64, BF, seed=35, causal=True, k_offsets=lens, cap=30.0)
    _check(dev, 1, 520, 520, 40, 2050, 128, BF, seed=36, causal=True)      # rows too few to be dealt out
    _check(dev, 1, 2048, 1, 10, 2050, 64, BF, seed=37, causal=True)        # one head: every part its own


def test_more_heads_than_workgroups_at_once(dev):
    _check(dev, 1, 800, 800, 33, 2020, 64, BF, seed=27, back=False, causal=True, offsets=[0, 3, 33],
           k_offsets=[0, 1000, 2020])


def test_masked_values_of_blocks_in_pieces(dev):
    """Infinities and NaN in keys of no document change no bit."""
    q, k, v, _, _ = (t.to(dev) for t in _inputs(1, 8, 8, 2200, 2200, 64, BF, 28))
    off = torch.tensor([0, 50, 2150], dtype=torch.int32, device=dev)
    want = attention_masked(q, k, v, 0.125, offsets=off, return_lse=True)
    k[:, :, 2150:], v[:, :, 2150:] = math.nan, math.inf
    v[:, :, 2160:] = math.nan
    got = attention_masked(q, k, v, 0.125, offsets=off, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_tokens(dev):
    for B, M, N in ((0, 4, 4), (2, 0, 5), (2, 5, 0)):
        q = torch.randn(B, 4, M, 64, device=dev, dtype=BF, requires_grad=True)
        k = torch.randn(B, 2, N, 64, device=dev, dtype=BF, requires_grad=True)
        v = torch.randn(B, 2, N, 64, device=dev, dtype=BF, requires_grad=True)
        o, lse = attention_masked(q, k, v, 0.125, causal=True, return_lse=True)
        assert o.shape == q.shape and not o.any() and (lse == -math.inf).all()
        for t, g in zip((q, k, v), torch.autograd.grad(o, (q, k, v), torch.ones_like(o))):
            assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("D", [64, 128])
def test_strides(dev, D):
    """Rows of a fused projection, odd row strides, misaligned bases, broadcast keys."""
    B, H, Hk, T = 2, 4, 2, 90
    g = torch.Generator(device=dev).manual_seed(0)
    rows = torch.randn(B, T, (H + 2 * Hk) * D + 3, generator=g, device=dev).to(BF)
    fused = rows[..., :(H + 2 * Hk) * D].unflatten(-1, (H + 2 * Hk, D)).transpose(1, 2)
    q, k, v = fused[:, :H], fused[:, H:H + Hk], fused[:, H + Hk:]
    want = attention_masked(q.contiguous(), k.contiguous(), v.contiguous(), 0.1, causal=True)
    got = attention_masked(q, k, v, 0.1, causal=True)                     # rows not 16-byte aligned
    assert torch.equal(got, want)
    qr = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = attention_masked(qr, k, v, 0.1, causal=True)
    assert torch.equal(got, want) and got.stride() == qr.stride()
    one = k[:1, :1]
    b = one.expand(B, Hk, T, D)
    want = attention_masked(q, b.contiguous(), b.contiguous(), 0.1)
    assert torch.equal(attention_masked(q, b, b, 0.1), want)
    leaf = one.detach().clone().requires_grad_()
    full = b.contiguous().detach().requires_grad_()
    d_o = torch.randn(q.shape, generator=g, device=dev).to(BF)
    e = leaf.expand(B, Hk, T, D)
    got, = torch.autograd.grad(attention_masked(q, e, e, 0.1), leaf, d_o)
    gk, = torch.autograd.grad(attention_masked(q, full, full, 0.1), full, d_o)
    want = gk.double().sum((0, 1), keepdim=True)
    # four bf16 gradients added in bf16: three sums and four values, each rounded
    assert ((got.double() - want).abs() <= 8 * 2.0 ** -8 * gk.double().abs().sum((0, 1), keepdim=True)).all()
    # d_o in another order than q
    turned = d_o.transpose(1, 2).contiguous().transpose(1, 2)
    a = torch.autograd.grad(attention_masked(q, full, full, 0.1), full, turned)[0]
    assert torch.equal(a, gk)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_no_row_may_see(dev, bad, dt):
    """NaN and infinities in padding, in another document and behind a causal
    query reach nobody who does not see them, forward and backward."""
    off = [3, 50, 120, 180]
    B, H, Hk, T, D = 1, 2, 1, 200, 64
    q, k, v, d_o, _ = _inputs(B, H, Hk, T, T, D, dt, 8)
    ref = masked_attention(q, k, v, D ** -0.5, causal=True, offsets=off, d_o=d_o, u=torch.finfo(dt).eps / 2)
    for name, at in (("padding", [0, 2, 180, 199]), ("document", [60]), ("future", [100])):
        qp, kp, vp, gp = (t.clone() for t in (q, k, v, d_o))
        for t in (qp, kp, vp, gp):
            t[:, :, at] = bad
        x = [t.to(dev).requires_grad_() for t in (qp, kp, vp)]
        o = attention_masked(*x, D ** -0.5, causal=True, offsets=torch.tensor(off, dtype=torch.int32, device=dev))
        dq, dk, dv = torch.autograd.grad(o, x, gp.to(dev))
        first = at[0] if name != "padding" else T
        doc_end = 120 if name != "padding" else T
        clean = torch.ones(T, dtype=torch.bool)                            # rows that see no bad value
        clean[first:doc_end] = False
        if name == "padding":
            clean[:3] = clean[180:] = False
            assert not o[:, :, ~clean.to(dev)].any()
        else:
            assert not torch.isfinite(o[:, :, at].float()).any()
        _near("o", o[:, :, clean.to(dev)], ref.o[:, :, clean], ref.o_bound[:, :, clean], dt)
        # a bad row reaches the gradients of the keys it sees, which are its document's earlier ones,
        # and a bad key its document's later rows
        out = clean.clone()
        if name != "padding":
            out[50:120] = False
        for n, got, want, bound in (("dk", dk, ref.dk, ref.dk_bound), ("dv", dv, ref.dv, ref.dv_bound)):
            _near(n, got[:, :, out.to(dev)], want[:, :, out], bound[:, :, out], dt)
        _near("dq", dq[:, :, clean.to(dev)], ref.dq[:, :, clean], ref.dq_bound[:, :, clean], dt)


def test_masked_value_beside_a_seen_infinity(dev):
    """A row that does see an infinite value gets it, by its sign."""
    q = torch.zeros(1, 1, 3, 64, dtype=BF, device=dev)
    v = torch.ones(1, 1, 3, 64, dtype=BF, device=dev)
    v[0, 0, 1, 0], v[0, 0, 1, 1], v[0, 0, 2, 1], v[0, 0, 2, 2] = math.inf, -math.inf, math.inf, math.nan
    o = attention_masked(q, q, v, 0.125, causal=True)[0, 0].float().cpu()
    assert (o[0] == 1).all()
    assert o[1, 0] == math.inf and o[1, 1] == -math.inf and (o[1, 2:] == 1).all()
    assert o[2, 0] == math.inf and math.isnan(o[2, 1]) and math.isnan(o[2, 2]) and (o[2, 3:] == 1).all()


def test_sharp_scores(dev):
    """Rows whose largest score lies far above the first tile's, and far below
    fp16's range of weights."""
    for dt, std in ((BF, 9.0), (HF, 9.0)):
        q, k, v, d_o, _ = _inputs(1, 2, 2, 130, 500, 64, dt, 21, std=std)
        k[:, :, 400] = 6 * q[:, :, 7]
        ref = masked_attention(q, k, v, 0.125, u=torch.finfo(dt).eps / 2)
        o = attention_masked(q.to(dev), k.to(dev), v.to(dev), 0.125)
        _near("o", o, ref.o, ref.o_bound, dt)


@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_fp16_gradients_keep_their_bits(dev, size):
    """Output gradients from far below to near fp16's range: dS is scaled before
    it is rounded."""
    q, k, v, d_o, _ = _inputs(1, 2, 1, 700, 700, 64, HF, 5)
    d_o = (d_o.float() * size).half()
    ref = masked_attention(q, k, v, 0.125, causal=True, d_o=d_o, u=2.0 ** -11)
    x = [t.to(dev).requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(attention_masked(*x, 0.125, causal=True), x, d_o.to(dev))
    for name, g, want in zip("qkv", got, ref[2:5]):
        rel = ((g.cpu().double() - want).norm() / want.norm()).item()
        # results of about size / 30: subnormal steps of 2^-24 where size is 1e-4
        assert rel <= 2 * 2.0 ** -11 + (2.0 ** -25 * math.sqrt(want.numel()) / want.norm().item()), (name, rel)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M", [1, 40])
def test_many_small_weights(dev, M, dt):
    """20,000 keys at 2^-15 to 2^-17 of the first one's weight, subnormal in fp16, together
    outweigh a third of it."""
    q, k, v, _, _ = _inputs(1, 1, 1, M, 20_000, 64, dt, 42, std=0.0)
    q[..., 0], k[..., 0] = 8.0, -torch.rand(20_000, dtype=torch.float64).to(dt) * 1.4 - 10.4
    k[:, :, 0, 0] = 0.0
    ref = masked_attention(q, k, v, 0.125, u=torch.finfo(dt).eps / 2)
    o, lse = attention_masked(q.to(dev), k.to(dev), v.to(dev), 0.125, return_lse=True)
    _near("o", o, ref.o, ref.o_bound, dt)
    assert ((lse.cpu().double() - ref.lse).abs() <= ref.lse_bound).all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_of_sharp_weights(dev, D, dt):
    """Scores with a spread of 6: dP - delta cancels, so delta has to come from more than
    the rounded output.  dS and the result are rounded once each, by 0.425 u of a
    norm (values spread evenly over a binade's logarithm): 0.60 u together, where
    delta from the rounded output adds 0.8 u."""
    u = torch.finfo(dt).eps / 2
    q, k, v, d_o, _ = _inputs(1, 2, 2, 600, 600, D, dt, 41, std=math.sqrt(6.0))
    x = [t.to(dev).requires_grad_() for t in (q, k, v)]
    for kw in (dict(), dict(slopes=torch.tensor([0.5, 0.1]))):
        ref = masked_attention(q, k, v, D ** -0.5, causal=True, d_o=d_o, u=u, **kw)
        o = attention_masked(*x, D ** -0.5, causal=True, **{n: t.to(dev) for n, t in kw.items()})
        for name, g, want in zip("qk", torch.autograd.grad(o, x, d_o.to(dev)), ref[2:4]):
            rel = ((g.cpu().double() - want).norm() / want.norm()).item()
            assert rel <= 0.75 * u, (name, rel / u)


def test_other_stream_and_graph(dev):
    """Captured forward and backward, replayed on new inputs between eager calls."""
    off = torch.tensor([0, 100, 260], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    make = lambda: torch.randn(1, 2, 260, 64, generator=g, device=dev).to(BF)  # noqa: E731
    x, d_o = [make().requires_grad_() for _ in range(3)], make()

    def step():
        o = attention_masked(*x, 0.125, causal=True, offsets=off, cap=30.0)
        return [o.detach(), *torch.autograd.grad(o, x, d_o)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        with torch.no_grad():
            for t in x:
                t.copy_(make())
            off[1] = 100 + 30 * turn
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), turn
    assert len(first) == 4


def test_gradients_by_differences(dev):
    """The oracle's own gradients, against differences of its output."""
    q, k, v, d_o, d_lse = _inputs(1, 2, 1, 6, 9, 64, BF, 1)
    q, k, v, d_o = (t.double() for t in (q, k, v, d_o))
    kw = dict(cap=3.0, slopes=torch.tensor([0.3, 0.1]), causal=True, prefix=2)

    def loss():
        r = masked_attention(q, k, v, 0.125, **kw)
        return (r.o * d_o).sum() + (r.lse * d_lse).sum()
    ref = masked_attention(q, k, v, 0.125, d_o=d_o, d_lse=d_lse, **kw)
    for t, want in ((q, ref.dq), (k, ref.dk), (v, ref.dv)):
        for at in (0, 77, t.numel() - 1):
            flat, eps = t.view(-1), 1e-5
            flat[at] += eps
            up = loss()
            flat[at] -= 2 * eps
            down = loss()
            flat[at] += eps
            assert abs((up - down) / (2 * eps) - want.reshape(-1)[at]) < 1e-7


def test_gradients_need_what_the_forward_kept(dev):
    from merging import _native
    q = torch.randn(1, 2, 9, 64, device=dev, dtype=BF, requires_grad=True)
    for kept in ((False, False), (True, False), (False, True)):
        with pytest.raises(RuntimeError, match="gradients need"):
            _native.attn_masked(q, q, q, 0.125, 0.0, None, False, None, 0, None, None, kept[0], False, kept[1])


def test_op_checks(dev):
    off = torch.tensor([0, 20, 50], dtype=torch.int32, device=dev)
    q = torch.randn(1, 4, 50, 64, device=dev, dtype=BF, requires_grad=True)
    k = torch.randn(1, 50, 2, 64, device=dev, dtype=BF).transpose(1, 2).requires_grad_()
    torch.library.opcheck(torch.ops.gpa.attn_masked.default,
                          (q, k, k, 0.125, 20.0, None, True, None, 3, off, off, True, True, True))
    from merging import _native
    d = q.detach()
    o, lse, rest = _native.attn_masked(d, k.detach(), k.detach(), 0.125, 0.0, None, False, None, 0, None, None, True,
                                       False, True)
    torch.library.opcheck(torch.ops.gpa.attn_masked_bwd.default,
                          (d, None, d, k.detach(), k.detach(), o, rest, lse, 0.125, 0.0, None, False, None, 0, None, None))

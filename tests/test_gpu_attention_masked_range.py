"""`attention_masked` and `attention_shared_prefix` where scores, values and
positions lie at the ends of their ranges, against the 64-bit definition.  Tolerances
are the oracle's elementwise bounds, as in test_gpu_attention_masked.py."""
import pytest
import torch

from merging.fused_attention import attention_masked, attention_shared_prefix
from oracle.masked_attention import masked_attention
from test_gpu_attention_masked import BF, HF, _check, _inputs, _near
from test_gpu_attention_shared_prefix import _check as _check_prefix

pytestmark = pytest.mark.gpu


# --- slopes below zero: scores grow with the distance --------------------------

DOWN = torch.tensor([-0.05, -0.25, 0.3, -2.0])


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,N,kw", [
    (700, 700, dict()),                              # later keys lie further from the first rows
    (700, 700, dict(causal=True, prefix=650)),
    (700, 700, dict(cap=20.0)),
    (300, 150, dict()),                              # rows that stand before their first key
    (40, 2000, dict(k_offsets=[0, 1990])),
    (3, 2000, dict(causal=True)),                    # few rows, the keys split
])
def test_slopes_below_zero(dev, M, N, kw, D, dt):
    offsets = [0, M] if "k_offsets" in kw else None
    _check(dev, 1, 4, 2, M, N, D, dt, seed=M + D, slopes=DOWN, offsets=offsets, **kw)


@pytest.mark.parametrize("dt,D", [(BF, 64), (HF, 128)])
def test_slopes_below_zero_in_cut_blocks(dev, D, dt):
    slopes = -torch.rand(8, generator=torch.Generator().manual_seed(3))
    _check(dev, 1, 8, 8, 2100, 2100, D, dt, seed=51, causal=True, prefix=1900, slopes=slopes)
    _check(dev, 1, 8, 8, 2100, 2100, D, dt, seed=52, offsets=[0, 600, 2050], slopes=slopes)


@pytest.mark.parametrize("dt,D", [(BF, 64), (HF, 128)])
def test_slopes_below_zero_over_a_shared_prefix(dev, D, dt):
    _check_prefix(dev, 3, 4, 2, 2, 3000, 70, D, dt, [70, 2, 33], slopes=DOWN)
    _check_prefix(dev, 2, 4, 2, 40, 700, 200, D, dt, [200, 41], slopes=DOWN)


# --- values near the end of bf16's range ----------------------------------------

@pytest.mark.parametrize("M,N", [(1, 500), (40, 500), (2, 20_000), (200, 3000)])
def test_large_values(dev, M, N):
    """Weights grow by 2^60 over a row's tiles, which an offset that stays where the first
    tile put it allows; times values of 1e25 that passes fp32."""
    q, k, v, _, _ = _inputs(1, 2, 1, M, N, 64, BF, 61, std=0.0)
    q[..., 0], k[:, :, 128:, 0] = 8.0, 42.0
    k[:, :, :128, 0] = torch.rand(128, generator=torch.Generator().manual_seed(1)).to(BF)
    for big in (v * 1e25, torch.full_like(v, 3e38)):
        ref = masked_attention(q, k, big, 0.125)
        o, lse = attention_masked(q.to(dev), k.to(dev), big.to(dev), 0.125, return_lse=True)
        _near("o", o, ref.o, ref.o_bound, BF)
        assert ((lse.cpu().double() - ref.lse).abs() <= ref.lse_bound).all()


def test_large_values_in_cut_blocks(dev):
    q, k, v, _, _ = _inputs(1, 8, 8, 2100, 2100, 64, BF, 62, std=0.0)
    q[..., 0], k[:, :, 128:, 0] = 8.0, 42.0
    v = v * 1e25
    ref = masked_attention(q, k, v, 0.125, causal=True)
    o = attention_masked(q.to(dev), k.to(dev), v.to(dev), 0.125, causal=True)
    _near("o", o, ref.o, ref.o_bound, BF)


# --- caps far above and below the scores -------------------------------------------

@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e12])
def test_caps_far_above_the_scores(dev, cap, D, dt):
    """Bounds from the uncapped scores, so that they do not grow with the cap.  The
    capped score's polynomial is off by 2.2 f of it and rounded six times, beside the
    product's D + 8 >= 72 f of no less: an eighth more."""
    q, k, v, d_o, d_lse = _inputs(2, 4, 2, 150, 150, D, dt, 71)
    kw = dict(causal=True, slopes=torch.tensor([0.5, 0.0, 0.03, 2.0]), d_o=d_o, d_lse=d_lse, u=torch.finfo(dt).eps / 2)
    ref, free = (masked_attention(q, k, v, D ** -0.5, cap=c, **kw) for c in (cap, None))
    x = [t.to(dev).requires_grad_() for t in (q, k, v)]
    o, lse = attention_masked(*x, D ** -0.5, cap=cap, causal=True, slopes=kw["slopes"].to(dev), return_lse=True)
    assert ((lse.detach().cpu().double() - ref.lse).abs() <= 1.125 * free.lse_bound).all()
    got = [o, *torch.autograd.grad([o, lse], x, [d_o.to(dev), d_lse.to(dev)])]
    for name in ("o", "dq", "dk", "dv"):
        want, loose, bound = (getattr(r, n) for r, n in ((ref, name), (free, name), (free, name + "_bound")))
        _near(name, got[("o", "dq", "dk", "dv").index(name)], want, 1.125 * bound + (want - loose).abs(), dt)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [100.0, 200.0, 2000.0])
def test_caps_that_scores_reach(dev, cap, D, dt):
    """Rows of scores from far below to far above the cap, beside each other."""
    q, k, v, d_o, _ = _inputs(1, 4, 2, 150, 150, D, dt, 73)
    q = (q.float() * torch.logspace(-2, 2, 150)[:, None]).to(dt)
    ref = masked_attention(q, k, v, D ** -0.5, cap=cap, d_o=d_o, u=torch.finfo(dt).eps / 2)
    x = [t.to(dev).requires_grad_() for t in (q, k, v)]
    o = attention_masked(*x, D ** -0.5, cap=cap)
    got = [o, *torch.autograd.grad(o, x, d_o.to(dev))]
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        _near(name, t, getattr(ref, name), getattr(ref, name + "_bound"), dt)


@pytest.mark.parametrize("M", [5, 150])
@pytest.mark.parametrize("cap", [1e-4, 1e-8, 1e-30])
def test_caps_far_below_the_scores(dev, cap, M):
    """Scores of plus or minus the cap, and of zero where a query or key is zero."""
    q, k, v, d_o, _ = _inputs(1, 2, 1, M, 150, 64, BF, 72)
    q[:, :, ::3], k[:, :, :40] = 0, 0
    ref = masked_attention(q, k, v, 0.125, cap=cap, d_o=d_o)
    x = [t.to(dev).requires_grad_() for t in (q, k, v)]
    o = attention_masked(*x, 0.125, cap=cap)
    got = [o, *torch.autograd.grad(o, x, d_o.to(dev))]
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        _near(name, t, getattr(ref, name), getattr(ref, name + "_bound"), BF)


# --- positions above 2^24 -----------------------------------------------------------

def test_documents_behind_2_24_tokens(dev):
    """A document behind 2^24 tokens of none: distances are its own, so results and
    gradients are those of the document alone, bit by bit."""
    far, D = 2 ** 24, 64
    g = torch.Generator(device=dev).manual_seed(81)
    short = [torch.randn(1, h, 320, D, generator=g, device=dev).to(BF) for h in (2, 1, 1, 2)]
    slopes = torch.tensor([0.5, 0.03], device=dev)

    def step(q, k, v, d_o, at):
        x = [t.requires_grad_() for t in (q, k, v)]
        off = torch.tensor([at, at + 3, at + 320], dtype=torch.int32, device=dev)
        o = attention_masked(*x, 0.125, causal=True, slopes=slopes, offsets=off)
        return [o.detach(), *torch.autograd.grad(o, x, d_o)]

    def behind(t):
        out = torch.zeros(1, far + 320, t.shape[1], D, dtype=BF, device=dev).transpose(1, 2)
        out[:, :, far:] = t
        return out
    want = step(*(t.clone() for t in short), 0)
    for name, got, ref in zip(("o", "dq", "dk", "dv"), step(*(behind(t) for t in short), far), want):
        assert torch.equal(got[:, :, far:], ref), name
        assert not got[:, :, :far].any(), name


@pytest.mark.parametrize("dt,D", [(BF, 64), (HF, 128)])
@pytest.mark.parametrize("H,Hk", [(6, 2), (5, 1), (40, 1), (64, 1), (100, 1)])
def test_slopes_of_head_groups_astride_row_tiles(dev, H, Hk, D, dt):
    slopes = torch.rand(H, generator=torch.Generator().manual_seed(H)) * 0.3
    _check(dev, 1, H, Hk, 77, 130, D, dt, seed=H, slopes=slopes, offsets=[0, 20, 77], k_offsets=[3, 60, 130])


# --- rows that overlap ----------------------------------------------------------------

def test_windows_that_slide_over_a_sequence(dev):
    """Queries, keys and values whose rows overlap, fewer of them than features."""
    g = torch.Generator(device=dev).manual_seed(91)
    t = torch.randn(3, 200, generator=g, device=dev).to(BF)
    q, k, v = (x.unfold(0, 64, 1)[:40].expand(1, 2, 40, 64).requires_grad_() for x in t)
    d_o = torch.randn(1, 2, 40, 64, generator=g, device=dev).to(BF)

    def step(*x):
        o = attention_masked(*x, 0.125, causal=True)
        return [o.detach(), *torch.autograd.grad(o, x, d_o)]
    plain = [x.detach().contiguous().requires_grad_() for x in (q, k, v)]
    assert all(torch.equal(a, b) for a, b in zip(step(q, k, v), step(*plain)))


# --- fp16 gradients beside infinite ones ------------------------------------------------

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1e-4, 300.0])
@pytest.mark.parametrize("lean", [1 / 128, 128.0])
def test_small_fp16_gradients_beside_an_infinite_one(dev, lean, size, D):
    """dS is scaled by a wave's largest value before it is rounded: of the finite ones.  An
    infinite output gradient at row 100 reaches the keys up to 100, in the middle of
    a block, and that row's dq; the others keep their accuracy.  Large keys (or
    queries) bring what small dS make well above fp16's smallest step."""
    q, k, v, d_o, _ = _inputs(1, 2, 1, 200, 200, D, HF, 95)
    q, k, v, d_o = q * lean, k / lean, v / 64, d_o * size
    ref = masked_attention(q, k, v, D ** -0.5, causal=True, d_o=d_o, u=2.0 ** -11)
    d_o[:, :, 100, 5] = float("inf")
    x = [t.to(dev).requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(attention_masked(*x, D ** -0.5, causal=True), x, d_o.to(dev))
    rows = torch.arange(200) != 100
    _near("dq", dq[:, :, rows.to(dev)], ref.dq[:, :, rows], ref.dq_bound[:, :, rows], HF)
    for name, got, want, bound in (("dk", dk, ref.dk, ref.dk_bound), ("dv", dv, ref.dv, ref.dv_bound)):
        _near(name, got[:, :, 101:], want[:, :, 101:], bound[:, :, 101:], HF)
    assert not torch.isfinite(dq[:, :, 100]).any() and not torch.isfinite(dk[:, :, :101]).any()
    # in norm: P and dS rounded and the result, with its subnormal steps
    for got, want in ((dq[:, :, rows.to(dev)], ref.dq[:, :, rows]), (dk[:, :, 101:], ref.dk[:, :, 101:])):
        rel = ((got.cpu().double() - want).norm() / want.norm()).item()
        assert rel <= 2 * 2.0 ** -11 + 2.0 ** -25 * want.numel() ** 0.5 / want.norm().item(), rel


# --- bases inside 16 bytes -------------------------------------------------------------

def test_contiguous_operands_behind_odd_bases(dev):
    g = torch.Generator(device=dev).manual_seed(97)
    size = 2 * 30 * 64
    flat = torch.randn(4, size + 8, generator=g, device=dev).to(BF)
    at = lambda i: [x[i:i + size].view(1, 2, 30, 64) for x in flat]  # noqa: E731

    def step(q, k, v, d_o):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        o = attention_masked(*x, 0.125, causal=True)
        shared = attention_shared_prefix(q, k[0], v[0], k, v, 0.125)
        return [o.detach(), shared, *torch.autograd.grad(o, x, d_o)]
    for i in (1, 4):
        assert all(t.is_contiguous() for t in at(i))
        assert all(torch.equal(a, b) for a, b in zip(step(*at(i)), step(*(t.clone() for t in at(i)))))

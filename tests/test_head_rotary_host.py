"""Refusals of `qk_norm_rotate`, `rotate_heads` and their C entry points, and the
frequency tables; none of this needs a GPU."""
import ctypes
import math

import pytest
import torch

from merging import _native
from merging.fused_rotary import RotaryAxes, qk_norm_rotate, rotary_axes, rotate_heads

FAKE = 4096
INV, UNS, WSP = _native.GPA_E_INVALID, _native.GPA_E_UNSUPPORTED, _native.GPA_E_WORKSPACE


def _fields(struct, base, kw):
    out = struct()
    for name, x in {**base, **kw}.items():
        setattr(out, name, x)
    return out


def _args(**kw):
    base = dict(q=FAKE, k=FAKE, B=2, N=3, H=4, Hk=2, D=64, pairs=32, positions=FAKE, freqs=FAKE, axes=FAKE,
                sections_count=2, s0=20, s1=12, norm=1, eps=1e-6)
    base.update({f"{t}_{s}": n for t in "qk" for s, n in (("sb", 768), ("sh", 64), ("sn", 256))})
    return _fields(_native._RotaryArgs, base, kw)


COMMON = [
    (dict(dtype=3), INV), (dict(dtype=-1), INV), (dict(dtype=1, pdtype=2), INV), (dict(dtype=0, pdtype=1), INV),
    (dict(B=-1), INV), (dict(N=-1), INV), (dict(H=-1), INV), (dict(Hk=-2), INV), (dict(D=-2), INV), (dict(pairs=-1), INV),
    (dict(D=0), UNS), (dict(D=63), UNS), (dict(D=258), UNS), (dict(D=62), INV), (dict(pairing=3), INV), (dict(pairing=-1), INV),
    (dict(sections_count=0), INV), (dict(sections_count=9), INV), (dict(s0=21), INV), (dict(s0=-1, s1=33), INV),
    (dict(s0=2 ** 31 - 1, s1=2 ** 31 - 1), INV), (dict(norm=3), INV), (dict(norm=-1), INV), (dict(eps=-1.0), INV),
    (dict(eps=math.nan), INV), (dict(eps=math.inf), INV), (dict(B=1 << 20, N=1 << 20), UNS), (dict(N=1 << 31), UNS),
    (dict(H=2048), UNS), (dict(Hk=2048), UNS), (dict(q=None), INV), (dict(k=None), INV), (dict(positions=None), INV),
    (dict(freqs=None), INV), (dict(axes=None), INV), (dict(positions_kind=3), INV), (dict(norm=0, q_w=FAKE), INV),
]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(q_out=None), INV), (dict(k_out=None), INV)])
def test_forward_argument_errors(kw, code):
    kw = dict(kw)
    dt, pdt, qo, ko = kw.pop("dtype", 1), kw.pop("pdtype", None), kw.pop("q_out", FAKE), kw.pop("k_out", FAKE)
    rc = _native.lib().gpa_head_rotary(dt, dt if pdt is None else pdt, ctypes.byref(_args(**kw)), qo, 768, 64, 256, ko, 384,
                                       64, 128, None)
    assert rc == code and _native.lib().gpa_last_error()


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(g=dict(dq=None)), INV), (dict(g=dict(dk=None)), INV), (dict(q_w=None), INV), (dict(k_w=None), INV),
    (dict(q_b=None), INV), (dict(k_b=None), INV), (dict(g=dict(d_q_out=None)), INV), (dict(g=dict(d_k_out=None)), INV),
    (dict(N=0), INV), (dict(B=0), INV), (dict(ws=None), WSP), (dict(ws_bytes=64), WSP), (dict(ws=FAKE + 8), WSP),
])
def test_backward_argument_errors(kw, code):
    kw = {**dict(q_w=FAKE, k_w=FAKE, q_b=FAKE, k_b=FAKE), **kw}
    dt, pdt = kw.pop("dtype", 1), kw.pop("pdtype", None)
    ws, ws_bytes = kw.pop("ws", FAKE), kw.pop("ws_bytes", 1 << 24)
    g = _fields(_native._RotaryGrads, {n: FAKE for n in "d_q_out d_k_out dq dk dq_w dk_w dq_b dk_b".split()}, kw.pop("g", {}))
    rc = _native.lib().gpa_head_rotary_bwd(dt, dt if pdt is None else pdt, ctypes.byref(_args(**kw)), ctypes.byref(g), ws,
                                           ws_bytes, None)
    assert rc == code and _native.lib().gpa_last_error()


def test_null_arguments_and_no_rows():
    L = _native.lib()
    assert L.gpa_head_rotary(1, 1, None, FAKE, 0, 0, 0, FAKE, 0, 0, 0, None) == INV
    assert L.gpa_head_rotary_bwd(1, 1, ctypes.byref(_args()), None, FAKE, 1 << 24, None) == INV
    none = _native._RotaryGrads()
    assert L.gpa_head_rotary_bwd(1, 1, ctypes.byref(_args()), ctypes.byref(none), None, 0, None) == 0
    for kw in (dict(B=0), dict(N=0), dict(H=0, Hk=0)):
        assert L.gpa_head_rotary(1, 1, ctypes.byref(_args(**kw)), None, 0, 0, 0, None, 0, 0, 0, None) == 0
    assert L.gpa_head_rotary_bwd_workspace_bytes(0, 3, 4, 2, 64, 1) == 0


@pytest.mark.parametrize("B,N,H,Hk", [(1, 1, 1, 1), (8, 1, 16, 4), (2, 8192, 32, 8), (1, 10_000, 1, 2000), (1, 10_000, 2000, 1)])
def test_workspace_stays_below_its_stated_size(B, N, H, Hk):
    """1,026 partials of two rows at most."""
    assert _native.lib().gpa_head_rotary_bwd_workspace_bytes(B, N, H, Hk, 128, 1) <= 1026 * 2 * 128 * 4


Q = torch.zeros(2, 4, 3, 16, dtype=torch.bfloat16)
POS = torch.zeros(3, 2, dtype=torch.int32)
ROT = rotary_axes((3, 5), device="cpu")


@pytest.mark.parametrize("kw,match", [
    (dict(kind="batch"), "kind"), (dict(eps=-1.0), "eps"), (dict(eps=1e300), "eps"), (dict(positions=None), "positions"),
    (dict(rotary=None), "positions"), (dict(rotary=ROT._replace(pairing="odd")), "pairing"),
    (dict(q=Q[0]), "expects"), (dict(k=Q[0]), "expects"),
    (dict(q_weight=torch.zeros(15, dtype=torch.bfloat16)), "GPU"),
])
def test_python_refusals(kw, match):
    a = {**dict(q=Q, k=Q, positions=POS, rotary=ROT), **kw}
    with pytest.raises(ValueError, match=match):
        qk_norm_rotate(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("rotary"), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=Q.double()), "dtype"), (dict(k=Q.float()), "one type"), (dict(k=Q[:1]), "one type"), (dict(k=Q[:, :, :2]), "one type"),
    (dict(freqs=ROT.freqs.float()), "fp64"), (dict(axes=ROT.axes.long()), "int32"), (dict(axes=ROT.axes[:3]), "int32"),
    (dict(freqs=None), "together"), (dict(sections=[3, 4]), "sections"), (dict(sections=[]), "sections"),
    (dict(sections=[-1, 9]), "sections"), (dict(sections=[1] * 8 + [0]), "sections"), (dict(positions=POS.short()), "positions"),
    (dict(positions=POS[:2]), "positions"), (dict(positions=POS[:, :1]), "positions"), (dict(positions=POS[None]), "positions"),
    (dict(freqs=torch.zeros(9, dtype=torch.float64), axes=torch.zeros(9, dtype=torch.int32)), "fit"), (dict(pairing=7), "pairing"),
    (dict(params=(torch.zeros(15, dtype=torch.bfloat16), None, None, None)), "parameters"),
    (dict(params=(torch.zeros(16, dtype=torch.float16), None, None, None)), "parameters"),
    (dict(params=(torch.zeros(16), torch.zeros(16, dtype=torch.bfloat16), None, None)), "parameters"),
])
def test_op_refusals(kw, match):
    a = {**dict(q=Q, k=Q, positions=POS, freqs=ROT.freqs, axes=ROT.axes, pairing=0, sections=[3, 5],
                params=(None,) * 4), **kw}
    with pytest.raises(ValueError, match=match):
        _native._rotary_check("x", *a.values())


def test_head_dims_are_refused():
    for D in (0, 15, 258):
        x = torch.zeros(1, 1, 1, D)
        with pytest.raises(NotImplementedError, match="head dim"):
            rotate_heads(x, POS[:1], ROT)
        with pytest.raises(NotImplementedError, match="head dim"):
            qk_norm_rotate(x, x, None, None)


def test_constants_have_no_gradient():
    with pytest.raises(ValueError, match="constants"):
        rotate_heads(Q, POS.float().requires_grad_(), ROT)


@pytest.mark.parametrize("kw", [dict(sections=()), dict(sections=(1,) * 9), dict(sections=(3, -1)), dict(ladder="log"),
                                dict(pairing="odd"), dict(order="random"), dict(pairing="blocks", order="dealt"),
                                dict(base=0.0), dict(base=math.inf), dict(base=-3.0)])
def test_tables_refuse(kw):
    with pytest.raises(ValueError, match="rotary_axes"):
        rotary_axes(kw.pop("sections", (4, 4)), device="cpu", **kw)


def test_tables():
    t = rotary_axes((2, 0, 3), base=32.0, device="cpu")
    assert t.axes.tolist() == [0, 0, 2, 2, 2] and t.sections == (2, 0, 3) and t.freqs.dtype == torch.float64
    assert torch.allclose(t.freqs, torch.tensor([32.0 ** (-j / 5) for j in range(5)], dtype=torch.float64), rtol=1e-15, atol=0)
    t = rotary_axes((2, 3), base=9.0, ladder="own", order="dealt", pairing="interleaved", device="cpu")
    assert t.axes.tolist() == [0, 1, 0, 1, 1]
    assert torch.allclose(t.freqs, torch.tensor([1, 1, 9 ** -0.5, 9 ** (-1 / 3), 9 ** (-2 / 3)], dtype=torch.float64), rtol=1e-15, atol=0)
    assert isinstance(t, RotaryAxes) and rotary_axes((0,), device="cpu").freqs.numel() == 0

"""Refusals of `norm_gate_residual` and its C entry points, none of which needs a
GPU."""
import ctypes

import pytest
import torch

from merging import _native
from merging.fused_norms import _gate_rows, norm_gate_residual

FAKE = 4096
INV, UNS, WSP = _native.GPA_E_INVALID, _native.GPA_E_UNSUPPORTED, _native.GPA_E_WORKSPACE


def _args(**kw):
    out = _native._NormArgs()
    for name, x in {**dict(x=FAKE, y=FAKE, gate=FAKE, w1=FAKE, b1=FAKE, w2=FAKE, b2=FAKE, stats=FAKE, rows=12,
                           C=64, groups=3, x_sn=64, y_sn=64, scale=1.0, eps=1e-6), **kw}.items():
        setattr(out, name, x)
    return out


COMMON = [
    (dict(dtype=3), INV), (dict(dtype=-1), INV), (dict(dtype=1, pdtype=2), INV), (dict(dtype=0, pdtype=1), INV),
    (dict(rows=-1), INV), (dict(C=-1), INV), (dict(groups=0), INV), (dict(groups=5), INV),
    (dict(C=0), UNS), (dict(C=8193), UNS), (dict(rows=3 << 30), UNS),
    (dict(eps=-1.0), INV), (dict(eps=float("nan")), INV), (dict(scale=float("inf")), INV),
    (dict(x=None), INV), (dict(y=None), INV), (dict(w2=None), INV), (dict(w1=None), INV),
]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(h=None), INV), (dict(out=None), INV), (dict(stats=FAKE + 4), INV)])
def test_forward_argument_errors(kw, code):
    kw = dict(kw)
    dt, pdt, h, out = kw.pop("dtype", 1), kw.pop("pdtype", None), kw.pop("h", FAKE), kw.pop("out", FAKE)
    rc = _native.lib().gpa_norm_gate(dt, dt if pdt is None else pdt, ctypes.byref(_args(**kw)), h, 64, out, 64, None)
    assert rc == code and _native.lib().gpa_last_error()


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(g=dict(dx=None)), INV), (dict(g=dict(dy=None)), INV), (dict(stats=None), INV), (dict(gate=None), INV),
    (dict(b1=None), INV), (dict(b2=None), INV), (dict(rows=0), INV), (dict(ws=None), WSP), (dict(ws_bytes=64), WSP),
    (dict(ws=FAKE + 8), WSP),
])
def test_backward_argument_errors(kw, code):
    kw = dict(kw)
    dt, pdt = kw.pop("dtype", 1), kw.pop("pdtype", None)
    ws, ws_bytes = kw.pop("ws", FAKE), kw.pop("ws_bytes", 1 << 24)
    g = _native._NormGrads()
    for name, x in {**{n: FAKE for n in "dh dout dx dy dgate dw1 db1 dw2 db2".split()}, **kw.pop("g", {})}.items():
        setattr(g, name, x)
    rc = _native.lib().gpa_norm_gate_bwd(dt, dt if pdt is None else pdt, ctypes.byref(_args(**kw)), ctypes.byref(g),
                                         ws, ws_bytes, None)
    assert rc == code and _native.lib().gpa_last_error()


def test_null_arguments_and_no_rows():
    L = _native.lib()
    assert L.gpa_norm_gate(1, 1, None, FAKE, 64, FAKE, 64, None) == INV
    assert L.gpa_norm_gate_bwd(1, 1, ctypes.byref(_args()), None, FAKE, 1 << 24, None) == INV
    assert L.gpa_norm_gate(1, 1, ctypes.byref(_args(rows=0)), None, 64, None, 64, None) == 0
    assert L.gpa_norm_gate_bwd_workspace_bytes(0, 64, 1) == 0


X = torch.zeros(2, 5, 64)


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(kind="batch"), ValueError, "kind"),
    (dict(eps=-1e-6), ValueError, "eps"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(gate=torch.zeros(5, 64)), ValueError, "gate"),
    (dict(gate=torch.zeros(1, 5, 64)), ValueError, "gate"),
    (dict(gate=torch.zeros(2, 1, 32)), ValueError, "gate"),
    (dict(gate=torch.zeros(1, 2, 1, 64)), ValueError, "gate"),
])
def test_norm_gate_residual_refuses(kw, err, text):
    with pytest.raises(err, match=text):
        norm_gate_residual(X, X, torch.ones(64), **kw)


def test_norm_gate_residual_refuses_shapes():
    with pytest.raises(ValueError, match="differ"):
        norm_gate_residual(X, X[:1], torch.ones(64))
    with pytest.raises(NotImplementedError, match="features"):
        norm_gate_residual(torch.zeros(1, 8193), torch.zeros(1, 8193), torch.ones(8193))


@pytest.mark.parametrize("kw,text", [
    (dict(y=X.bfloat16()), "differ"), (dict(x=X.double(), y=X.double()), "dtype"),
    (dict(w1=torch.ones(63)), "post_weight"), (dict(w2=torch.ones(64).bfloat16()), "parameters"),
    (dict(w1=torch.ones(64).half()), "parameters"), (dict(b1=torch.ones(64)), "post_bias"),
    (dict(gate=torch.zeros(3, 64)), "gate"), (dict(gate=torch.zeros(0, 64)), "gate"),
])
def test_op_refuses(kw, text):
    a = {**dict(x=X, y=X, w1=None, b1=None, gate=None, w2=torch.ones(64), b2=None), **kw}
    with pytest.raises(ValueError, match=text):
        _native._norm_check("x", *a.values())


def test_gate_rows():
    assert _gate_rows(X, torch.zeros(64)).shape == (1, 64)
    assert _gate_rows(X, torch.zeros(1, 1, 64)).shape == (1, 64)
    assert _gate_rows(X, torch.zeros(2, 1, 64)).shape == (2, 64)
    assert _gate_rows(X, torch.zeros(2, 5, 64)).shape == (10, 64)

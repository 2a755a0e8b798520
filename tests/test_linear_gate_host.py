"""Refusals of `linear_gate_residual` and its C entry points; none of this needs a GPU."""
import ctypes

import pytest
import torch

from merging import _native
from merging.fused_linear import linear_gate_residual

FAKE = 4096
INV, UNS, WSP = _native.GPA_E_INVALID, _native.GPA_E_UNSUPPORTED, _native.GPA_E_WORKSPACE


def _fields(struct, base, kw):
    out = struct()
    for name, x in {**base, **kw}.items():
        setattr(out, name, x)
    return out


def _args(**kw):
    return _fields(_native._LinearArgs, dict(x=FAKE, w=FAKE, bias=FAKE, gate=FAKE, residual=FAKE, M=300, N=64, K=128, x_s=128,
                                             w_s=128, residual_s=64, act=1), kw)


COMMON = [
    (dict(dtype=0), INV), (dict(dtype=3), INV), (dict(dtype=1, pdtype=2), INV), (dict(dtype=2, pdtype=1), INV), (dict(M=-1), INV),
    (dict(N=-1), INV), (dict(K=-8), INV), (dict(act=-1), INV), (dict(act=5), INV), (dict(x=None), INV), (dict(w=None), INV),
    (dict(M=1 << 30), UNS), (dict(N=1 << 30), UNS), (dict(K=1 << 21), UNS),
]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(y=None), INV), (dict(z=FAKE + 4), INV), (dict(z_dtype=1), INV)])
def test_forward_argument_errors(kw, code):
    kw = dict(kw)
    dt, pdt, y, z, zdt = kw.pop("dtype", 1), kw.pop("pdtype", None), kw.pop("y", FAKE), kw.pop("z", FAKE), kw.pop("z_dtype", 0)
    rc = _native.lib().gpa_linear_gate(dt, dt if pdt is None else pdt, ctypes.byref(_args(**kw)), y, 64, z, zdt, FAKE, 1 << 30, None)
    assert rc == code and _native.lib().gpa_last_error()


@pytest.mark.parametrize("kw,least", [
    (dict(M=70, N=70, K=80_000, x_s=80_000, w_s=80_000), 2 * 70 * 72 * 4),      # a sum that is cut has parts
    (dict(K=127), (300 + 64) * 128 * 2), (dict(M=3, K=127), (3 + 64) * 128 * 2),  # padded copies of x and w
    (dict(x=FAKE + 8), 300 * 128 * 2), (dict(w_s=130), 64 * 128 * 2), (dict(x_s=1 << 21), 300 * 128 * 2), (dict(w_s=-128), 64 * 128 * 2),
    (dict(K=0), (300 + 64) * 8 * 2)])
def test_forward_workspace(kw, least):
    L, a = _native.lib(), _args(**kw)
    need = L.gpa_linear_gate_workspace_bytes(ctypes.byref(a))
    assert need >= least
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 8, need)):
        assert L.gpa_linear_gate(1, 1, ctypes.byref(a), FAKE, 70, None, 0, ws, size, None) == WSP


def test_calls_without_a_workspace():
    L = _native.lib()
    for kw in (dict(M=16), dict(M=1, x_s=3), dict(M=0), dict(N=0), dict(M=-1)):
        assert L.gpa_linear_gate_workspace_bytes(ctypes.byref(_args(**kw))) == 0
    assert L.gpa_linear_gate_workspace_bytes(None) == 0


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(g=dict(dy=None)), INV), (dict(g=dict(z=None)), INV), (dict(act=0, g=dict(z=None)), INV), (dict(gate=None), INV),
    (dict(g=dict(z=FAKE + 4)), INV), (dict(g=dict(z_dtype=1)), INV), (dict(K=0), INV),
    (dict(M=0), INV), (dict(N=0), INV), (dict(N=1 << 21), UNS), (dict(ws=None), WSP), (dict(ws_bytes=64), WSP), (dict(ws=FAKE + 8), WSP),
])
def test_backward_argument_errors(kw, code):
    kw = dict(kw)
    dt, pdt, ws, ws_bytes = kw.pop("dtype", 1), kw.pop("pdtype", None), kw.pop("ws", FAKE), kw.pop("ws_bytes", 1 << 40)
    g = _fields(_native._LinearGrads, dict(dy=FAKE, z=FAKE, dx=FAKE, dw=FAKE, dbias=FAKE, dgate=FAKE, dy_s=64, dx_s=128, dw_s=128), kw.pop("g", {}))
    rc = _native.lib().gpa_linear_gate_bwd(dt, dt if pdt is None else pdt, ctypes.byref(_args(**kw)), ctypes.byref(g), ws, ws_bytes, None)
    assert rc == code and _native.lib().gpa_last_error()


def test_nothing_to_do():
    L = _native.lib()
    none = _native._LinearGrads()
    assert L.gpa_linear_gate(1, 1, None, FAKE, 64, None, 0, None, 0, None) == INV
    assert L.gpa_linear_gate_bwd(1, 1, ctypes.byref(_args()), None, FAKE, 1 << 30, None) == INV
    assert L.gpa_linear_gate_bwd(1, 1, ctypes.byref(_args()), ctypes.byref(none), None, 0, None) == 0
    for kw in (dict(M=0), dict(N=0)):
        assert L.gpa_linear_gate(1, 1, ctypes.byref(_args(**kw)), None, 64, None, 0, None, 0, None) == 0


X, W = torch.zeros(5, 16, dtype=torch.bfloat16), torch.zeros(7, 16, dtype=torch.bfloat16)
B = torch.zeros(7, dtype=torch.bfloat16)


@pytest.mark.parametrize("kw,match", [
    (dict(activation="tanh"), "activation"), (dict(weight=W[:, :8]), "go together"), (dict(weight=B), "go together"),
    (dict(residual=torch.zeros(5, 8)), "residual"), (dict(residual=torch.zeros(7)), "residual"), (dict(), "GPU"),
])
def test_python_refusals(kw, match):
    a = {**dict(weight=W), **kw}
    with pytest.raises(ValueError, match=match):
        linear_gate_residual(X, a.pop("weight"), **a)
    with pytest.raises(NotImplementedError, match="float64"):
        linear_gate_residual(X.double(), W)


@pytest.mark.parametrize("kw,match", [
    (dict(x=X.float()), "bf16 or fp16"), (dict(w=W.half()), "one type"), (dict(x=X[0]), "one type"), (dict(bias=B[:6]), "bias"),
    (dict(gate=B[None]), "gate"), (dict(bias=B.half()), "bias and gate"), (dict(bias=B.float(), gate=B), "bias and gate"),
    (dict(residual=X), "residual"), (dict(residual=torch.zeros(5, 7)), "residual"), (dict(act=5), "activation"),
])
def test_op_refusals(kw, match):
    a = {**dict(x=X, w=W, bias=None, gate=None, residual=None, act=0), **kw}
    with pytest.raises(ValueError, match=match):
        _native._linear_check("y", *a.values())


@pytest.mark.parametrize("M", [1, 16])
@pytest.mark.parametrize("K", [8, 8192])
def test_too_many_columns_of_few_rows(M, K):
    """More than 2^32 threads, which a launch does not have."""
    a = _args(M=M, N=(1 << 26) + 1, K=K, x_s=K, w_s=K)
    assert _native.lib().gpa_linear_gate(1, 1, ctypes.byref(a), FAKE, 1 << 27, None, 0, None, 0, None) == UNS


def test_kept_sums_are_fp32():
    L, a = _native.lib(), _args(act=1)
    for zdt in (_native._DTYPE_CODES[torch.bfloat16], _native._DTYPE_CODES[torch.float16]):
        assert L.gpa_linear_gate(1, 1, ctypes.byref(a), FAKE, 64, FAKE, zdt, FAKE, 1 << 30, None) == INV
        g = _fields(_native._LinearGrads, dict(dy=FAKE, z=FAKE, dx=FAKE, dy_s=64, dx_s=128, z_dtype=zdt), {})
        assert L.gpa_linear_gate_bwd(1, 1, ctypes.byref(a), ctypes.byref(g), FAKE, 1 << 40, None) == INV
    assert torch.ops.gpa.linear_gate.default(X.to("meta"), W.to("meta"), None, None, None, 1, True)[1].dtype == torch.float32

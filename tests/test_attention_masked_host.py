"""Refusals of the masked attention's entry points, none of which needs a GPU:
the C ABI's codes before any device work, and the Python functions' errors."""
import ctypes

import pytest
import torch

from merging import _native
from merging.fused_attention import attention_masked, attention_shared_prefix

FAKE = 4096     # a 16-byte aligned non-null address; validation returns before any use
INV, UNS, WSP = _native.GPA_E_INVALID, _native.GPA_E_UNSUPPORTED, _native.GPA_E_WORKSPACE


def _args(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=FAKE, B=2, H=4, Hk=2, M=10, N=10, D=64,
             q_sb=2560, q_sh=640, q_sm=64, k_sb=1280, k_sh=640, k_sn=64, v_sb=1280, v_sh=640, v_sn=64,
             o_sb=2560, o_sh=640, o_sm=64, lse_sb=40, lse_sh=10, docs=1, sm_scale=0.125)
    a.update(kw)
    out = _native._MaskedArgs()
    for name, x in a.items():
        setattr(out, name, x)
    return out


def _forward(dtype=_native.GPA_DTYPE_BF16, ws=None, ws_bytes=0, **kw):
    return _native.lib().gpa_attn_masked(dtype, ctypes.byref(_args(**kw)), ws, ws_bytes, None)


COMMON = [
    (dict(M=-1), INV), (dict(P=-1), INV), (dict(docs=0), INV), (dict(dtype=0), INV),
    (dict(D=32), UNS), (dict(D=256), UNS), (dict(Hk=3), INV), (dict(Hk=0), INV),
    (dict(sm_scale=0.0), INV), (dict(sm_scale=float("nan")), INV), (dict(sm_scale=float("inf")), INV),
    (dict(cap=-1.0), INV), (dict(cap=float("inf")), INV),
    (dict(docs=2), INV), (dict(docs=2, q_offsets=FAKE), INV), (dict(docs=2, k_offsets=FAKE), INV),
    (dict(lens=FAKE, k_offsets=FAKE), INV),
    (dict(prefix_len=3), INV), (dict(prefix=FAKE), INV), (dict(prefix_len=-1, causal=1), INV),
    (dict(q=None), INV), (dict(k=None), INV), (dict(v=None), INV), (dict(o=None), INV),
    (dict(q=FAKE + 8), INV), (dict(k_sn=68), INV), (dict(q_sh=644), INV), (dict(o_sm=66), INV),
    (dict(k_sn=1 << 23), UNS), (dict(v_sn=-64), UNS),
    (dict(M=1 << 30), UNS), (dict(N=1 << 30), UNS), (dict(B=1 << 28), UNS),
]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(P=10, pk=FAKE, pv=FAKE, q_offsets=FAKE, k_offsets=FAKE), INV),
    (dict(P=10, pk=FAKE), INV), (dict(P=10, pk=FAKE, pv=FAKE, pk_sn=4), INV),
    (dict(P=10, pk=FAKE, pv=FAKE, pk_sn=64, pv_sn=64, pk_sh=640, pv_sh=640), WSP),
    (dict(N=100_000), WSP),
])
def test_forward_argument_errors(kw, code):
    assert _forward(**kw) == code
    assert _native.lib().gpa_last_error()


def test_null_arguments_and_workspace_alignment():
    L = _native.lib()
    assert L.gpa_attn_masked(1, None, None, 0, None) == INV
    need = L.gpa_attn_masked_workspace_bytes(2, 4, 2, 10, 100_000, 0, 64)
    assert need > 0 and _forward(N=100_000, ws=FAKE + 4, ws_bytes=need) == WSP
    assert _forward(N=100_000, ws=FAKE, ws_bytes=need - 1) == WSP
    assert L.gpa_attn_masked_workspace_bytes(2, 4, 2, 10, 10, 0, 64) == 0
    assert L.gpa_attn_masked_bwd_workspace_bytes(2, 4, 2, 10) == 2 * 2 * 1 * 256 * 4


def test_rest_of_the_output_is_aligned():
    assert _forward(o_rest=FAKE + 8) == INV
    assert _native.lib().gpa_last_error()


def test_workspaces_of_blocks_in_pieces():
    """Sized for any mask of the sizes; a call asks for what its own mask needs."""
    L = _native.lib()
    big = dict(B=1, H=8, Hk=8, M=4096, N=4096, q_sb=0, k_sb=0, v_sb=0, o_sb=0, q_sh=4096 * 64, k_sh=4096 * 64,
               v_sh=4096 * 64, o_sh=4096 * 64, q_sm=64, k_sn=64, v_sn=64, o_sm=64)
    need = L.gpa_attn_masked_workspace_bytes(1, 8, 8, 4096, 4096, 0, 64)
    assert need > 0
    assert _forward(ws=FAKE, ws_bytes=need - 1, causal=1, **big) == WSP
    assert _forward(ws=FAKE, ws_bytes=0, causal=1, **big) == WSP
    rec = 8 * (4096 // 64) * 256 * 4
    need = L.gpa_attn_masked_bwd_workspace_bytes(1, 8, 8, 4096)
    assert need > rec
    shape = dict(do_sb=0, do_sh=4096 * 64, do_sm=64, dq_sb=0, dq_sh=4096 * 64, dq_sm=64, dk_sb=0, dk_sh=4096 * 64,
                 dk_sn=64, dv_sb=0, dv_sh=4096 * 64, dv_sn=64)
    assert _backward(ws_bytes=need - 1, g=shape, lse=FAKE, causal=1, **big) == WSP


def test_nothing_to_do_is_ok():
    assert _forward(B=0) == 0 and _forward(M=0) == 0


def _backward(dtype=_native.GPA_DTYPE_BF16, ws=FAKE, ws_bytes=1 << 20, grads=True, g=None, **kw):
    out = _native._MaskedGrads()
    for name, x in {**dict(d_o=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, do_sb=2560, do_sh=640, do_sm=64, dq_sb=2560,
                           dq_sh=640, dq_sm=64, dk_sb=1280, dk_sh=640, dk_sn=64, dv_sb=1280, dv_sh=640,
                           dv_sn=64), **(g or {})}.items():
        setattr(out, name, x)
    return _native.lib().gpa_attn_masked_bwd(dtype, ctypes.byref(_args(**kw)),
                                             ctypes.byref(out) if grads else None, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(grads=False), INV), (dict(lse=None), INV), (dict(g=dict(d_o=None)), INV), (dict(g=dict(dk=None)), INV),
    (dict(g=dict(dq=FAKE + 2)), INV), (dict(g=dict(do_sm=65)), INV), (dict(lens=FAKE), UNS),
    (dict(P=10, pk=FAKE, pv=FAKE, pk_sn=64, pv_sn=64), UNS), (dict(q_sh=1 << 29), UNS),
    (dict(g=dict(do_sm=1 << 25)), UNS), (dict(ws=None), WSP), (dict(ws_bytes=100), WSP), (dict(M=0), INV),
])
def test_backward_argument_errors(kw, code):
    assert _backward(**kw) == code
    assert _native.lib().gpa_last_error()


def _qkv(dt=torch.bfloat16, M=6, N=6, D=64, H=4, Hk=2):
    return torch.zeros(2, H, M, D, dtype=dt), torch.zeros(2, Hk, N, D, dtype=dt), torch.zeros(2, Hk, N, D, dtype=dt)


I32 = torch.int32


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(sm_scale=0.0), ValueError, "sm_scale"),
    (dict(sm_scale=float("nan")), ValueError, "sm_scale"),
    (dict(cap=0.0), ValueError, "cap"),
    (dict(cap=float("inf")), ValueError, "cap"),
    (dict(prefix=3), ValueError, "causal"),
    (dict(prefix=-1, causal=True), ValueError, "negative"),
    (dict(offsets=torch.zeros(1, dtype=I32)), ValueError, "docs"),
    (dict(k_offsets=torch.zeros(3, dtype=I32)), ValueError, "queries"),
    (dict(slopes=torch.zeros(4, requires_grad=True)), ValueError, "slopes"),
])
def test_attention_masked_refuses(kw, err, text):
    kw = dict(kw)
    scale = kw.pop("sm_scale", 0.125)
    with pytest.raises(err, match=text):
        attention_masked(*_qkv(), scale, **kw)


def test_attention_masked_refuses_shapes_and_types():
    q, k, v = _qkv(M=5)
    with pytest.raises(ValueError, match="k_offsets"):
        attention_masked(q, k, v, 0.125, offsets=torch.tensor([0, 5], dtype=I32))
    with pytest.raises(NotImplementedError, match="float64"):
        attention_masked(*_qkv(torch.float64), 0.125)
    with pytest.raises(ValueError, match="expects"):
        attention_masked(q[0], k, v, 0.125)


@pytest.mark.parametrize("q,k,v", [
    ((2, 4, 6, 64), (2, 3, 6, 64), (2, 3, 6, 64)),
    ((2, 4, 6, 64), (2, 2, 6, 64), (2, 2, 5, 64)),
    ((2, 4, 6, 64), (1, 2, 6, 64), (1, 2, 6, 64)),
    ((2, 4, 6, 64), (2, 2, 6, 128), (2, 2, 6, 128)),
    ((2, 4, 6, 64), (2, 0, 6, 64), (2, 0, 6, 64)),
])
def test_shapes_that_do_not_match(q, k, v):
    with pytest.raises(ValueError, match="multiple"):
        _native._masked_shapes("x", *(torch.zeros(s, dtype=torch.bfloat16) for s in (q, k, v)))


@pytest.mark.parametrize("t", [torch.zeros(4, dtype=torch.int64), torch.zeros(3, dtype=I32),
                               torch.zeros(3, 4, dtype=I32), torch.zeros(1, 1, 4, dtype=I32)])
def test_tables_that_do_not_match(t):
    with pytest.raises(ValueError, match="offsets must be"):
        _native._table("x", "offsets", t, 2, 4, I32)


def test_shared_prefix_refuses():
    q, k, v = _qkv()
    pk = torch.zeros(2, 9, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        attention_shared_prefix(q, pk, pk, k, v, 0.125)
    with pytest.raises(ValueError, match="sm_scale"):
        attention_shared_prefix(q, pk, pk, k, v, -1.0)
    with pytest.raises(NotImplementedError, match="float64"):
        attention_shared_prefix(q.double(), pk, pk, k, v, 0.125)

"""Refusals of `draft_tree`, `attention_tree` and their C entry points; none of this
needs a GPU."""
import ctypes

import pytest
import torch

from merging import _native
from merging.fused_attention import attention_tree, draft_tree

FAKE = 4096
INV, UNS, WSP = _native.GPA_E_INVALID, _native.GPA_E_UNSUPPORTED, _native.GPA_E_WORKSPACE


def _call(**kw):
    a = dict(q=FAKE, cache_k=FAKE, cache_v=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=FAKE, B=2, H=4, Hk=2, T=8, N=3000, D=64,
             q_sb=2048, q_sh=64, q_st=256, ck_sb=384_000, ck_sh=192_000, ck_sn=64, cv_sb=384_000, cv_sh=192_000, cv_sn=64,
             k_sb=1024, k_sh=512, k_st=64, v_sb=1024, v_sh=512, v_st=64, o_sb=2048, o_sh=64, o_st=256, lse_sb=32, lse_sh=8,
             lengths=FAKE, seen=FAKE, sm_scale=0.125, cap=0.0, dtype=1, ws=FAKE, ws_bytes=1 << 30)
    a.update(kw)
    dt, ws, ws_bytes = a.pop("dtype"), a.pop("ws"), a.pop("ws_bytes")
    out = _native._TreeArgs()
    for name, x in a.items():
        setattr(out, name, x)
    return _native.lib().gpa_attn_tree(dt, ctypes.byref(out), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), INV), (dict(dtype=3), INV), (dict(B=-1), INV), (dict(T=-1), INV), (dict(N=-1), INV), (dict(Hk=-1), INV),
    (dict(D=32), UNS), (dict(D=256), UNS), (dict(Hk=3), INV), (dict(Hk=0), INV), (dict(sm_scale=0.0), INV),
    (dict(sm_scale=float("nan")), INV), (dict(cap=-1.0), INV), (dict(T=1025), UNS), (dict(N=1 << 30), UNS),
    (dict(B=1 << 30), UNS), (dict(q=None), INV), (dict(cache_k=None), INV), (dict(cache_v=None), INV), (dict(k=None), INV),
    (dict(v=None), INV), (dict(o=None), INV), (dict(seen=None), INV), (dict(q=FAKE + 2), INV), (dict(k=FAKE + 8), INV),
    (dict(k_sb=1028), INV), (dict(v_sb=1028), INV), (dict(k_st=68), INV), (dict(ck_sn=68), INV), (dict(cv_sb=4), INV),
    (dict(o_st=4), INV), (dict(ck_sn=1 << 23), UNS), (dict(v_st=1 << 23), UNS), (dict(ck_sn=-64), UNS),
    (dict(ws=None), WSP), (dict(ws_bytes=64), WSP), (dict(ws=FAKE + 8), WSP),
    (dict(B=1 << 22, H=64, Hk=64, T=1, N=1), UNS), (dict(B=1 << 20, N=1 << 29, T=1, H=1, Hk=1), UNS),
])
def test_attention_argument_errors(kw, code):
    assert _call(**kw) == code and _native.lib().gpa_last_error()


def test_nothing_to_do():
    for kw in (dict(B=0), dict(T=0), dict(H=0, Hk=0)):
        assert _call(**{**kw, **{n: None for n in ("q", "k", "v", "o", "cache_k", "cache_v", "seen", "ws")}}) == 0
    assert _native.lib().gpa_attn_tree(1, None, FAKE, 64, None) == INV


@pytest.mark.parametrize("args,code", [
    ((FAKE, 8, FAKE, None, -1, 8, FAKE, FAKE), INV), ((FAKE, 8, FAKE, None, 2, -8, FAKE, FAKE), INV),
    ((FAKE, 8, FAKE, None, 2, 1025, FAKE, FAKE), UNS), ((FAKE, 8, FAKE, None, 1 << 23, 8, FAKE, FAKE), UNS),
    ((None, 8, FAKE, None, 2, 8, FAKE, FAKE), INV), ((FAKE, 8, None, None, 2, 8, FAKE, FAKE), INV),
    ((FAKE, 8, FAKE, None, 2, 8, None, FAKE), INV), ((FAKE, 8, FAKE, None, 2, 8, FAKE, None), INV),
    ((None, 8, None, None, 0, 8, None, None), 0), ((None, 8, None, None, 2, 0, None, None), 0),
])
def test_draft_argument_errors(args, code):
    assert _native.lib().gpa_draft_tree(*args, None) == code


@pytest.mark.parametrize("B,H,Hk,T,N,D", [(1, 8, 2, 26, 130_001, 64), (8, 32, 8, 64, 8192, 128), (64, 16, 16, 16, 4096, 64),
                                          (300, 8, 1, 4, 100_000, 64), (1, 1, 1, 1024, 1 << 29, 128), (1, 4, 4, 1, 200, 64)])
def test_workspace_stays_below_its_stated_size(B, H, Hk, T, N, D):
    """4 (D + 2) bytes a row and piece, of 768 / (key heads and blocks of 128 rows) pieces, or two
    for each sequence, and 4 a sequence."""
    R = T * (H // Hk)
    target = max(1, 768 // (Hk * -(-R // 128)))
    got = _native.lib().gpa_attn_tree_workspace_bytes(B, H, Hk, T, N, D)
    assert got <= 4 * (D + 2) * max(target, 2 * B) * Hk * R + 4 * (B + 1)
    assert N > 200 or got == 0


Q, K, C = (torch.zeros(2, h, n, 64, dtype=torch.bfloat16) for h, n in ((4, 5), (2, 5), (2, 30)))
SEEN, LEN = torch.zeros(2, 5, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


@pytest.mark.parametrize("kw,match", [
    (dict(k=K[:, :, :4], v=K[:, :, :4]), "drafted keys"), (dict(v=K[:, :1]), "multiple of Hk"), (dict(k=K.half()), "k is"),
    (dict(ck=C[:, :1]), "cache_k"), (dict(cv=C[:, :, :9]), "cache_v"), (dict(cv=C.half()), "cache_v"), (dict(ck=C[0]), "cache_k"),
    (dict(seen=SEEN[:, :4]), "seen"), (dict(seen=SEEN.long()), "seen"), (dict(seen=SEEN[..., 0]), "seen"),
    (dict(lengths=LEN.long()), "lengths"), (dict(lengths=LEN[:1]), "lengths"), (dict(lengths=LEN[None]), "lengths"),
    (dict(slopes=torch.zeros(3)), "slopes"), (dict(slopes=torch.zeros(4, dtype=torch.float64)), "slopes"),
])
def test_shapes_are_refused(kw, match):
    a = {**dict(q=Q, ck=C, cv=C, k=K, v=K, lengths=LEN, seen=SEEN, slopes=None), **kw}
    with pytest.raises(ValueError, match=match):
        _native._tree_check("x", *a.values())


def test_long_drafts_are_refused():
    q = torch.zeros(1, 1, 1025, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="1025"):
        _native._tree_check("x", q, C[:1, :1], C[:1, :1], q, q, None, SEEN, None)


def test_python_refusals():
    with pytest.raises(ValueError, match="GPU"):
        attention_tree(Q, C, C, K, K, 0.1, seen=SEEN)
    with pytest.raises(ValueError, match="GPU"):
        draft_tree(LEN[None].expand(2, 2), LEN)
    with pytest.raises(ValueError, match="sm_scale"):
        attention_tree(Q, C, C, K, K, 0.0, seen=SEEN)
    with pytest.raises(ValueError, match="cap"):
        attention_tree(Q, C, C, K, K, 0.1, seen=SEEN, cap=-1.0)
    with pytest.raises(ValueError, match="constants"):
        attention_tree(Q, C, C, K, K, 0.1, seen=SEEN, slopes=torch.zeros(4, requires_grad=True))
    with pytest.raises(NotImplementedError, match="float64"):
        attention_tree(Q.double(), C, C, K, K, 0.1, seen=SEEN)

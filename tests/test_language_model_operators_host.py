"""Arguments of the language-model operators at the ends of their ranges; none of this
needs a GPU."""
import math
import random

import pytest
import torch

from merging import _native
from merging.fused_attention import attention_masked, attention_shared_prefix
from merging.fused_norms import norm_gate_residual
from test_attention_masked_host import FAKE, _backward, _forward

BF = torch.bfloat16


@pytest.mark.parametrize("value", [1e-50, 1e-40, 1e39, 1e300])
def test_numbers_outside_fp32_are_refused(value):
    """The kernels take them in fp32, where a cap of 0 would be none at all."""
    q = torch.zeros(1, 2, 3, 64, dtype=BF)
    p = torch.zeros(2, 3, 64, dtype=BF)
    for call in (lambda s, c: attention_masked(q, q, q, s, cap=c),
                 lambda s, c: attention_shared_prefix(q, p, p, q, q, s, cap=c)):
        with pytest.raises(ValueError, match="cap"):
            call(0.125, value)
        with pytest.raises(ValueError, match="sm_scale"):
            call(value, None)
    x = torch.zeros(3, 8, dtype=BF)
    if value > 1:
        with pytest.raises(ValueError, match="eps"):
            norm_gate_residual(x, x, x[0], eps=value)
        for scale in (value, -value):
            with pytest.raises(ValueError, match="scale"):
                norm_gate_residual(x, x, x[0], scale=scale)
    else:
        with pytest.raises(ValueError, match="GPU"):         # 0 in fp32, as eps and scale may be
            norm_gate_residual(x, x, x[0], eps=value, scale=value)


@pytest.mark.parametrize("seed", range(40))
def test_workspaces_stay_below_their_stated_sizes(seed):
    """8 (D + 2) bytes for each of 98,304 (head dim 64) or 65,536 (128) rows and a list of
    66,000; over a shared prefix for each query and head, where they are more.  The
    backward: 101 MB, and 16 bytes for each query and head of whole 64-row tiles."""
    rng = random.Random(seed)
    L = _native.lib()
    D, hk, G = rng.choice([64, 128]), rng.choice([1, 2, 5, 8, 64]), rng.choice([1, 3, 4, 32])
    size = lambda top: int(math.exp(rng.uniform(0, math.log(top))))  # noqa: E731
    B, M, N, P = size(300), size(20_000), size(300_000), size(300_000)
    least = {64: 98_304, 128: 65_536}[D]
    each = 8 * (D + 2)
    assert L.gpa_attn_masked_workspace_bytes(B, hk * G, hk, M, N, 0, D) <= each * least + 66_000
    got = L.gpa_attn_masked_workspace_bytes(B, hk * G, hk, M, N, P, D)
    assert each * B * hk * G * M <= got <= each * max(least, B * hk * G * M) + 66_000
    tiles = B * hk * (-(-G * M // 64))
    assert L.gpa_attn_masked_bwd_workspace_bytes(B, hk * G, hk, M) <= 101_000_000 + 16 * 64 * tiles


@pytest.mark.parametrize("rows,step", [(40, 1), (100, 1), (40, 8), (1, 1)])
def test_results_of_overlapping_rows_have_rows(rows, step):
    """Windows that slide over a sequence: rows that overlap, in an order of their own."""
    t = torch.arange(4000.0).unfold(0, 64, step)[:rows].expand(2, 3, rows, 64)
    new = _native._like(t)
    assert new.shape == t.shape and new.stride(-1) == 1 and _native._rows_ok(new, 8)


@pytest.mark.parametrize("lens", [torch.zeros(0, 2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32),
                                  torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)])
def test_lengths_are_one_row(lens):
    q = torch.zeros(2, 2, 3, 64, dtype=BF)
    with pytest.raises(ValueError, match=r"lengths must be torch.int32 \[2\]"):
        _native._masked_args("x", q, q, q, q, None, 0.125, 0.0, None, True, lens=lens)


def test_launches_of_2_32_threads_are_refused():
    """A workgroup of 256 threads for each sequence and key head at least."""
    one = dict(H=1, Hk=1, M=1, N=1)
    assert _forward(B=1 << 24, **one) == _native.GPA_E_UNSUPPORTED
    assert _backward(B=1 << 24, **one) == _native.GPA_E_UNSUPPORTED
    # the join over a shared prefix: 64 threads a query and head
    assert _forward(B=4, H=2, Hk=2, M=1 << 24, N=1, P=10, pk=FAKE, pv=FAKE, pk_sn=64, pv_sn=64, pk_sh=640,
                    pv_sh=640) == _native.GPA_E_UNSUPPORTED


@pytest.mark.parametrize("at", [0, 1, 4])
def test_rows_behind_any_base_are_aligned(at):
    """A tensor that is contiguous but begins inside 16 bytes is copied too."""
    t = torch.arange(512.0).to(BF)[at:at + 384].view(1, 2, 3, 64)
    rows = _native._rows8(t)
    assert torch.equal(rows, t) and _native._rows_ok(rows, 8)

"""`norm_gate_residual` over very many rows."""
import pytest
import torch

from merging.fused_norms import norm_gate_residual

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_more_rows_than_one_grid_dimension(dev):
    """A width that is not a multiple of 8 takes a workgroup a row."""
    R, C = 2 ** 24 + 3, 7
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(5, C, generator=g, device=dev, dtype=BF)
    w = torch.randn(C, generator=g, device=dev, dtype=BF)
    want = norm_gate_residual(x, x, w, post_weight=w)
    many = x.repeat(R // 5 + 1, 1)[:R]
    for got, ref in zip(norm_gate_residual(many, many, w, post_weight=w), want):
        assert torch.equal(got, ref.repeat(R // 5 + 1, 1)[:R])

"""`attention_masked` and `attention_shared_prefix` where scores, values and
positions lie at the ends of their ranges, against the 64-bit definition.  Tolerances
are the oracle's elementwise bounds, as in test_gpu_attention_masked.py."""
import pytest
import torch

from merging.fused_attention import attention_masked
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

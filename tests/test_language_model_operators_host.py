"""Arguments of the language-model operators at the ends of their ranges; none of this
needs a GPU."""
import pytest
import torch

from merging.fused_attention import attention_masked, attention_shared_prefix
from merging.fused_norms import norm_gate_residual

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

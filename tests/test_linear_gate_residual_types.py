"""A residual of another type than 16-bit x is refused by `linear_gate_residual`: the result is of x's
type, to which a wider residual would be rounded."""
import pytest
import torch

from merging.fused_linear import linear_gate_residual

F, BF, HF = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("x,residual", [(BF, F), (HF, F), (BF, HF), (HF, BF), (BF, torch.float64)])
def test_other_types_are_refused(x, residual):
    x, r = torch.zeros(5, 16, dtype=x), torch.zeros(5, 7, dtype=residual)
    for grad in (False, True):
        with pytest.raises(ValueError, match="residual is torch"):
            linear_gate_residual(x, torch.zeros(7, 16, dtype=x.dtype), residual=r.clone().requires_grad_(grad))


@pytest.mark.gpu
@pytest.mark.parametrize("to", [BF, HF])
def test_types_that_are_taken(dev, to):
    """x's own; with an fp32 x, which is cast, any other is cast with it."""
    g = torch.Generator(device=dev).manual_seed(0)
    x, w, r = (torch.randn(*s, generator=g, device=dev).to(to) for s in ((5, 16), (8, 16), (5, 8)))
    want = linear_gate_residual(x, w, residual=r)
    assert want.dtype == to
    for res in (r, r.float()):
        with torch.autocast("cuda", dtype=to):
            assert torch.equal(linear_gate_residual(x.float(), w, residual=res), want)
    assert torch.equal(linear_gate_residual(x, w.float(), residual=r), want)
    with torch.autocast("cuda", dtype=to), pytest.raises(ValueError, match="residual is torch"):
        linear_gate_residual(x, w, residual=r.float())

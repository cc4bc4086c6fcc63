"""Newton-Schulz steps against their 64-bit definition, within bounds that do not follow the kernel's roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo
from muon_fixed_bounds import CASES, STEPS, allowed, gradient


@pytest.mark.parametrize("steps", STEPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize(dtype, steps):
    from haste_b200.optim import orthogonalize
    g = [gradient(*case).to(dtype).cuda() for case in CASES]
    for case, x, got in zip(CASES, g, orthogonalize(g, steps)):
        exact = eo.orthogonalize(x, steps)
        off = float((got.double() - exact).norm()) / float(exact.norm())
        assert off <= allowed(steps), (case, off)

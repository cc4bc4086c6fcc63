"""The model of the kernel's roundings, which other tests derive their bounds from, is itself within fixed bounds of the 64-bit definition."""
import pytest
import torch

from oracle import encoder_oracle as eo
from muon_fixed_bounds import CASES, STEPS, allowed, gradient


@pytest.mark.parametrize("kind,shape", CASES)
def test_model(kind, shape):
    g = gradient(kind, shape)
    for steps in STEPS:
        exact = eo.orthogonalize(g, steps)
        got = eo.orthogonalize_rounded(g, steps).float().to(torch.bfloat16).double()
        assert float((got - exact).norm()) <= allowed(steps) * float(exact.norm()), steps

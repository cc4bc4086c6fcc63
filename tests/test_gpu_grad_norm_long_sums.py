"""Gradient norm of so many elements that an fp32 sum over a thread's share would lose small values behind large ones."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do


@pytest.mark.parametrize("times", [1, 16])
def test_small_values_behind_large_ones(times):
    """A thread adds 64 squares at most before it goes on in 64 bits, then 8 sums, 5 times lanes and 8 warps are added: (64 + 8 + 5 + 8) U of the sum at
    worst, half of it of the root, whose own roundings are 2 U."""
    from haste_b200.optim import grad_norm
    big = torch.full((2 ** 31,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    big[:1000] = 16.0
    rest = torch.full((2 ** 31,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    want = math.sqrt(256000.0 + (2.0 ** 31 - 1000 + (times - 1) * 2.0 ** 31) * 2.0 ** -20)
    assert abs(float(grad_norm([big] + [rest] * (times - 1))) - want) <= want * (85 / 2 + 2) * do.U

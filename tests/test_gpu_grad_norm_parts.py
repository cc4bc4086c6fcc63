"""Gradient norm of more elements than one launch takes (2^38), the last launch a small one: the same tensor listed many times."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_small_rest_does_not_replace_the_sum():
    from haste_b200.optim import grad_norm
    big = torch.full((2 ** 31,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    small = torch.full((1000,), 16.0, device="cuda")
    want = math.sqrt(128 * 2.0 ** 11 + 256000.0)
    for grads in ([big] * 128 + [small], [small] + [big] * 128):
        assert abs(float(grad_norm(grads)) - want) <= 1e-6 * want

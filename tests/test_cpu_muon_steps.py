"""A number of Newton-Schulz steps that 32 bits do not hold is refused, not cut down to another number."""
import pytest
import torch


@pytest.mark.parametrize("steps", [2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1, -2 ** 32 + 5])
def test_steps_out_of_range(steps):
    from haste_b200.optim import muon_step, orthogonalize
    x = torch.zeros(4, 8)
    for call in (lambda: orthogonalize([x], steps), lambda: orthogonalize([], steps), lambda: muon_step([x], [x], x, step=1, steps=steps)):
        with pytest.raises(RuntimeError, match="steps=-?[0-9]+ is out of range"):
            call()


def test_steps_beyond_64_bits():
    from haste_b200.optim import orthogonalize
    with pytest.raises(OverflowError):
        orthogonalize([], 2 ** 70)
    assert orthogonalize([], 5) == []

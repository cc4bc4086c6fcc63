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


def test_workspace_of_few_rows():
    """Less than what larger matrices of that many rows and columns, rounded up to 64, would take."""
    import ctypes
    from haste_b200 import _lib
    i64 = lambda v: (ctypes.c_int64 * len(v))(*v)
    scratch = lambda rows, cols: _lib.lib.haste_muon_scratch(i64(rows), i64(cols), len(rows))
    for p in (1, 4, 5, 16, 17, 32):
        for q in (p, 64, 1000, 100000, 1 << 24):
            up = -(-max(p, q) // 64) * 64
            assert 8 * p * p <= scratch([p], [q]) == scratch([q], [p]) <= 2 * (3 * 64 * up + 64 * 64) + 4096
    assert scratch([32] * 2000, [512] * 2000) <= 1 << 30
    assert scratch([8, 600], [100, 1000]) <= scratch([8], [100]) + scratch([600], [1000])

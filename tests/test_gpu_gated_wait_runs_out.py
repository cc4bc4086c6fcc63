"""A wait in the block's products that runs out: the launch comes to an end by itself, the status is reported once, and the next call is right."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_wait_runs_out():
    """One tile of more than two milliseconds of products (2^20 features), and waits that give up after half of one."""
    from haste_b200 import _lib
    from haste_b200.feedforward import gated_forward
    D = 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)
    x, wg, wu, wd = r(40, D), r(64, D), r(64, D), r(8, 64)
    want = gated_forward(x, wg, wu, wd, keep=True)
    torch.cuda.synchronize()
    assert _lib.lib.haste_poll_status() == _lib.OK
    try:
        assert _lib.lib.haste_debug_set_wait_limit(1000) == _lib.OK
        gated_forward(x, wg, wu, wd)                                           # returns by itself; its result is not valid
        torch.cuda.synchronize()
    finally:
        _lib.lib.haste_debug_set_wait_limit(4_000_000_000)
    assert _lib.lib.haste_poll_status() == _lib.ERR_TIMEOUT and "wait id" in _lib.last_error()
    assert _lib.lib.haste_poll_status() == _lib.OK
    assert all(torch.equal(a, b) for a, b in zip(gated_forward(x, wg, wu, wd, keep=True), want))
    torch.cuda.synchronize()
    assert _lib.lib.haste_poll_status() == _lib.OK

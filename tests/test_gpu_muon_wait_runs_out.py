"""A wait in the Newton-Schulz steps that runs out: the launch comes to an end by itself, the status is reported once, weights stay as they were and results that are not complete are NaN; the next
call is right."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF = torch.bfloat16
# one tile a product; several (narrow tiles); many matrices of several shapes (wide tiles)
LISTS = [[(64, 64)], [(512, 768), (300, 260)], [(520, 300)] * 30 + [(257, 1030)] * 40 + [(64, 70)]]


@pytest.fixture
def short_waits():
    """From the call on, the waits of kernels that are launched then last half a microsecond, which no product takes."""
    from haste_b200 import _lib
    assert _lib.lib.haste_poll_status() == _lib.OK
    yield lambda: _lib.lib.haste_debug_set_wait_limit(1000)
    _lib.lib.haste_debug_set_wait_limit(4_000_000_000)


def _reported_once():
    from haste_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.lib.haste_debug_set_wait_limit(4_000_000_000) == _lib.OK
    assert _lib.lib.haste_poll_status() == _lib.ERR_TIMEOUT and "wait id" in _lib.last_error()
    assert _lib.lib.haste_poll_status() == _lib.OK


def _matrices(shapes, scale):
    gen = torch.Generator().manual_seed(len(shapes))
    return [scale * torch.randn(s, generator=gen).cuda() for s in shapes]


@pytest.mark.parametrize("shapes", LISTS)
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_weights_stay(shapes, dtype, short_waits):
    from haste_b200.optim import moment_offsets, muon_step
    g, w = _matrices(shapes, 1e-3), [x.to(dtype) for x in _matrices(shapes, 0.02)]
    before, at = [x.clone() for x in w], moment_offsets([x.numel() for x in w])
    short_waits()
    muon_step(w, g, torch.zeros(at[-1], device="cuda"), step=1, lr=0.1, stochastic_rounding=False)
    _reported_once()
    assert all(torch.equal(a, b) for a, b in zip(w, before))
    muon_step(w, g, torch.zeros(at[-1], device="cuda"), step=1, lr=0.1, weight_decay=0.0, stochastic_rounding=False)
    for new, old, u in zip(w, before, g):
        # (the first momentum is 0.05 of the gradient: the same direction)
        x, tol = eo.orthogonalize_bound(u)
        rate = eo.muon_rate(u.shape, 0.1, "original")
        want = old.double() - rate * x
        assert float((new.double() - want).norm()) <= rate * tol + eo.U * 8 * float(want.norm()) + torch.finfo(dtype).eps / 2 * float(want.norm())


@pytest.mark.parametrize("shapes", LISTS)
def test_results_are_nan(shapes, short_waits):
    from haste_b200.optim import orthogonalize
    g = _matrices(shapes, 1e-3)
    want = orthogonalize(g)
    short_waits()
    got = orthogonalize(g)
    _reported_once()
    assert all(x.isnan().all() for x in got)
    assert all(torch.equal(a, b) for a, b in zip(orthogonalize(g), want))

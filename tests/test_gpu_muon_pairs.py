"""Newton-Schulz steps make progress with however few pairs of blocks run at once: with one, and with more than the device holds, the rest of which start when others have ended."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def pairs():
    from haste_b200 import _lib
    yield lambda n: _lib.lib.haste_debug_set_product_pairs(n)
    assert _lib.lib.haste_debug_set_product_pairs(0) == _lib.OK


# one list in the narrow form, one in the wide form
@pytest.mark.parametrize("shapes", [[(64, 64)] * 40 + [(300, 520), (200, 130)] * 3, [(520, 300)] * 40 + [(257, 1030)] * 40 + [(64, 70)] * 60])
def test_any_number(shapes, pairs):
    from haste_b200 import _lib
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(0)
    g = [torch.randn(s, generator=gen).cuda() for s in shapes]
    want = orthogonalize(g)
    for n in (1, 2, 7, 74, 75, 200, 1000):
        assert pairs(n) == _lib.OK
        got = orthogonalize(g)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n
    torch.cuda.synchronize()
    assert _lib.lib.haste_poll_status() == _lib.OK


def test_beside_other_work(pairs):
    """Two lists and a product on three streams at once."""
    from haste_b200 import _lib
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(1)
    lists = [[torch.randn(400, 500, generator=gen).cuda() for _ in range(30)] for _ in range(2)]
    want = [orthogonalize(g) for g in lists]
    a = torch.randn(4096, 4096, device="cuda").bfloat16()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for n in (0, 150):
        assert pairs(n) == _lib.OK
        got = [None, None]
        for _ in range(3):
            with torch.cuda.stream(streams[2]):
                for _ in range(4):
                    a @ a
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i] = orthogonalize(lists[i])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for i in range(2) for x, y in zip(got[i], want[i]))
    assert _lib.lib.haste_poll_status() == _lib.OK

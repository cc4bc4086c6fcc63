"""The embedding's gradient where the device cannot place the cluster that sorts the tokens: several launches do, to the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo


@pytest.fixture
def largest_cluster():
    from haste_b200 import _lib
    yield lambda blocks: _lib.lib.haste_debug_set_cluster_limit(blocks)
    assert _lib.lib.haste_debug_set_cluster_limit(16) == _lib.OK


# sizes at which a cluster has 1, 2, 4, 8 and 16 blocks, with 1, 4 and 8 tokens a thread; passes of one digit to three
@pytest.mark.parametrize("tokens,rows", [(1, 1), (7, 300), (1024, 255), (1025, 256), (4097, 5003), (16384, 70000), (16385, 32000), (65537, 1000), (131072, 65536)])
def test_same_bits(tokens, rows, largest_cluster):
    from haste_b200 import _lib
    from haste_b200.embedding import embedding_backward
    gen = torch.Generator().manual_seed(tokens)
    ids = (torch.rand(tokens, generator=gen) ** 3 * (rows + 2)).long().sub_(1).cuda()         # some are no row
    dy = torch.randn(tokens, 24, generator=gen).cuda()
    want = embedding_backward(dy, ids, rows, 2.0, 0)
    exact, tol = eo.embedding_grad(dy, ids, rows, 2.0, 0)
    assert eo.outside(want, exact, tol) is None
    for blocks in (8, 4, 1, 0):
        assert largest_cluster(blocks) == _lib.OK
        assert torch.equal(embedding_backward(dy, ids, rows, 2.0, 0), want)


def test_in_a_graph(largest_cluster):
    from haste_b200.embedding import embedding_backward
    ids, dy = torch.randint(0, 500, (30, 200), device="cuda"), torch.randn(30, 200, 40, device="cuda").to(torch.bfloat16)
    want = embedding_backward(dy, ids, 500)
    largest_cluster(0)
    embedding_backward(dy, ids, 500)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = embedding_backward(dy, ids, 500)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)

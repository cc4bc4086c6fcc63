"""Tables whose rows share memory: one row expanded to many, overlapping windows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 7, 1])
def test_forward_and_gradient(D, dtype):
    from haste_b200.embedding import embedding, embedding_forward
    gen = torch.Generator().manual_seed(D)
    ids = torch.randint(0, 20, (6, 5), generator=gen).cuda()
    row, flat = torch.randn(D, generator=gen).to(dtype).cuda(), torch.randn(20 * D + D, generator=gen).to(dtype).cuda()
    for table in (row.expand(20, D), row.view(1, D).expand(20, D), flat.as_strided((20, D), (1, 1)), flat.as_strided((20, D), (max(1, D // 2), 1)), flat[:20].view(20, 1).expand(20, D)):
        assert torch.equal(embedding_forward(ids, table, 2.0), 2 * table[ids])
    leaf, dy = row.clone().requires_grad_(), torch.randint(-4, 5, (6, 5, D), generator=gen).to(dtype).cuda()
    (embedding(ids, leaf.expand(20, D)) * dy).sum().backward()
    # small whole numbers: sums without a rounding
    assert torch.equal(leaf.grad.float(), dy.float().sum((0, 1)))

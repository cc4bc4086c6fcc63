"""Embedding, gated block and Muon where places in a tensor pass 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF = torch.bfloat16
MANY, D = 2200000, 1024                # rows of more than 2^31 elements


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("60 GB of memory wanted")
    yield
    torch.cuda.empty_cache()


def test_embedding_of_many_tokens():
    from haste_b200.embedding import embedding_backward, embedding_forward
    gen = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 1000, (MANY,), generator=gen, device="cuda")
    table = torch.randn(1000, D, generator=gen, device="cuda").to(BF)
    y = embedding_forward(ids, table)
    for rows in (slice(0, 100), slice(MANY // 2, MANY // 2 + 100), slice(MANY - 100, MANY)):
        assert torch.equal(y[rows], table[ids[rows]])
    # small whole numbers: every sum is exact in any order
    dy = y.copy_(torch.randint(-4, 5, (MANY, D), generator=gen, device="cuda", dtype=torch.int8))
    want = torch.zeros(1000, D, device="cuda")
    for at in range(0, MANY, 200000):
        want.index_add_(0, ids[at:at + 200000], dy[at:at + 200000].float())
    assert torch.equal(embedding_backward(dy, ids, 1000, dtype=torch.float32), want)


def test_embedding_of_many_rows():
    from haste_b200.embedding import embedding_backward, embedding_forward
    gen = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.cat([torch.randint(0, MANY, (700,), generator=gen, device="cuda"), torch.tensor([0, MANY - 1, MANY - 1, 2 ** 21, MANY], device="cuda")])
    table = torch.randn(MANY, D, generator=gen, device="cuda", dtype=BF)
    y = embedding_forward(ids, table)
    assert torch.equal(y[:-1], table[ids[:-1]]) and y[-1].isnan().all()
    del table
    dy = torch.randint(1, 5, (ids.numel(), D), generator=gen, device="cuda").to(BF)
    got = embedding_backward(dy, ids, MANY)
    rows, back = torch.unique(ids[:-1], return_inverse=True)
    assert torch.equal(got[rows].float(), torch.zeros(rows.numel(), D, device="cuda").index_add_(0, back, dy[:-1].float()))
    assert torch.equal(got.any(1).nonzero().view(-1), rows)


def test_gated_block_of_many_rows():
    from haste_b200.feedforward import gated_backward, gated_forward
    T, width, hidden, out = 1100000, 16, 2048, 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF)
    x, wg, wu, wd = r(T, width), r(hidden, width) * 0.25, r(hidden, width) * 0.25, r(out, hidden) * 0.02
    dy = torch.zeros(T, out, device="cuda", dtype=BF)
    dy[-300:] = r(300, out)
    y, gate, up = gated_forward(x, wg, wu, wd, "silu", keep=True)
    for rows in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        for got, want, tol in zip((y, gate, up), *eo.gated(x[rows], wg, wu, wd, "silu")):
            assert eo.outside(got[rows], want, tol) is None
    grads = gated_backward(dy, x, wg, wu, wd, gate, up, "silu")
    last = slice(T - 300, T)               # the other rows' gradients are zeros
    for i, (want, tol) in enumerate(zip(*eo.gated_grad(dy[last], x[last], wg, wu, wd, gate[last], up[last], "silu"))):
        assert eo.outside(grads[i][last] if i == 0 else grads[i], want, tol) is None
    assert not grads[0][:-300].any()


def test_muon_of_many_elements():
    from haste_b200.optim import muon_step
    gen = torch.Generator(device="cuda").manual_seed(4)
    shape = (1024, 524288)
    params = [torch.randn(shape, generator=gen, device="cuda", dtype=BF) for _ in range(5)]
    grads = [torch.randn(shape, generator=gen, device="cuda", dtype=BF) for _ in range(2)]
    grads = [grads[i % 2] for i in range(5)]
    alone, momentum = params[4].clone(), torch.zeros(params[4].numel(), device="cuda")
    muon_step([alone], [grads[4]], momentum, step=1, lr=0.1, stochastic_rounding=False)
    every = torch.zeros(5 * params[4].numel(), device="cuda")
    muon_step(params, grads, every, step=1, lr=0.1, stochastic_rounding=False)
    assert torch.equal(params[4], alone) and torch.equal(every[-momentum.numel():], momentum)

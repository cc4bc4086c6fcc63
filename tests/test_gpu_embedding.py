"""Token embedding against the 64-bit oracle: types, ids that repeat a thousand times or never, padding, ids that are no row, odd widths, strides."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF, F32 = torch.bfloat16, torch.float32
# tokens, width, rows
SHAPES = [(1, 1, 1), (1, 768, 30), (9, 768, 3000), (300, 7, 5), (65, 64, 64), (1000, 1021, 333), (4099, 96, 5003), (5000, 8, 300), (20000, 40, 70000), (700, 4096, 50), (3, 9000, 4)]


def _ids(tokens, rows, kind, gen):
    if kind == "one":
        return torch.full((tokens,), rows // 2, dtype=torch.int64)
    if kind == "words":
        return (torch.exp(torch.rand(tokens, generator=gen, dtype=torch.float64) * torch.log(torch.tensor(rows + 1.0))) - 1).long().clamp(0, rows - 1)
    return torch.randint(0, rows, (tokens,), generator=gen)


def _check_grad(got, dy, ids, rows, scale, padding=None):
    want, tol = eo.embedding_grad(dy, ids, rows, scale, padding)
    assert got.shape == want.shape
    bad = eo.outside(got, want, tol, "dtable")
    assert bad is None, bad


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    from haste_b200.embedding import embedding_forward
    tokens, D, V = shape
    gen = torch.Generator().manual_seed(tokens + D)
    table = torch.randn(V, D, generator=gen).to(dtype).cuda()
    for wide, scale in ((torch.int64, 1.0), (torch.int32, 3.7)):
        ids = _ids(tokens, V, "words", gen).to(wide).cuda()
        y = embedding_forward(ids, table, scale)
        assert y.dtype == dtype and y.shape == (tokens, D)
        bad = eo.outside(y, *eo.embedding(ids, table, scale), "y")
        assert bad is None, bad
        if scale == 1.0:
            assert torch.equal(y, table[ids])


@pytest.mark.parametrize("types", [(BF, BF), (F32, F32), (BF, F32), (F32, BF)])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, types):
    from haste_b200.embedding import embedding_backward
    tokens, D, V = shape
    gen = torch.Generator().manual_seed(tokens * 3 + D)
    dy = torch.randn(tokens, D, generator=gen).to(types[0]).cuda()
    for kind in ("words", "even", "one"):
        ids = _ids(tokens, V, kind, gen).cuda()
        got = embedding_backward(dy, ids, V, 0.7, dtype=types[1])
        assert got.dtype == types[1]
        _check_grad(got, dy, ids, V, 0.7)
        assert torch.equal(got, embedding_backward(dy, ids.int(), V, 0.7, dtype=types[1]))            # and the same bits every time


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("padding", [0, 7, -1, 299])
def test_padding_and_ids_that_are_no_row(padding, dtype):
    from haste_b200.embedding import embedding_backward, embedding_forward
    gen = torch.Generator().manual_seed(5)
    ids = torch.randint(-3, 304, (2000,), generator=gen).cuda()
    dy, table = torch.randn(2000, 24, generator=gen).to(dtype).cuda(), torch.randn(300, 24, generator=gen).to(dtype).cuda()
    got = embedding_backward(dy, ids, 300, 1.0, padding)
    assert not got[padding].any()
    _check_grad(got, dy, ids, 300, 1.0, padding)
    y = embedding_forward(ids, table)
    wrong = (ids < 0) | (ids >= 300)
    assert wrong.any() and y[wrong].isnan().all() and torch.equal(y[~wrong], table[ids[~wrong]])
    huge = torch.tensor([2 ** 40, -2 ** 40, 5], device="cuda")
    assert embedding_forward(huge, table).isnan().any(1).tolist() == [True, True, False]
    _check_grad(embedding_backward(dy[:3], huge, 300), dy[:3], huge, 300, 1.0)


def test_frequent_words_among_many_tokens():
    """Rows whose tokens fill many blocks, one after the other, and rows that end at a block's border."""
    from haste_b200.embedding import embedding_backward
    gen = torch.Generator().manual_seed(9)
    counts = torch.tensor([64, 63, 1, 0, 0, 130, 62, 2000, 64, 64, 0, 5000, 1, 1])
    ids = torch.repeat_interleave(torch.arange(len(counts)), counts)
    ids = ids[torch.randperm(len(ids), generator=gen)].cuda()
    for dtype, D in ((F32, 1030), (BF, 1032)):
        dy = torch.randn(len(ids), D, generator=gen).to(dtype).cuda()
        _check_grad(embedding_backward(dy, ids, len(counts)), dy, ids, len(counts), 1.0)


def test_many_rows_and_few_tokens():
    from haste_b200.embedding import embedding_backward
    ids = torch.tensor([250000, 3, 250001, 3, 131072], device="cuda")
    dy = torch.randn(5, 16, device="cuda")
    got = embedding_backward(dy, ids, 250002)
    _check_grad(got, dy, ids, 250002, 1.0)
    assert int(got.any(1).sum()) == 4


@pytest.mark.parametrize("tokens", [1024, 1025, 2048, 2049, 16384, 16385, 65536, 65537, 131072, 131073, 200001])
def test_numbers_of_tokens_at_which_the_sort_changes(tokens):
    from haste_b200.embedding import embedding_backward
    gen = torch.Generator().manual_seed(tokens)
    for rows, kind in ((200, "words"), (70000, "even"), (300, "one")):
        ids = _ids(tokens, rows, kind, gen).cuda()
        dy = torch.randn(tokens, 12, generator=gen).cuda()
        got = embedding_backward(dy, ids, rows)
        _check_grad(got, dy, ids, rows, 1.0)
        assert torch.equal(got, embedding_backward(dy, ids, rows))


def test_strides_shapes_and_no_tokens():
    from haste_b200.embedding import embedding_backward, embedding_forward
    wide = torch.randn(50, 80, device="cuda")
    ids = torch.randint(0, 50, (6, 5), device="cuda")
    for table in (wide[:, 8:72], wide[:, 3:50], wide.t()[:50, :40], wide[::2][:, :64].repeat(2, 1)):
        y = embedding_forward(ids.t(), table)
        assert y.shape == (5, 6, table.shape[1]) and torch.equal(y, table[ids.t()])
    dy = torch.randn(6, 5, 200, device="cuda")
    for part in (dy[..., 8:72], dy[..., 1:70], dy[..., ::2], torch.randn(64, device="cuda").expand(6, 5, 64), torch.randn(6, 1, 64, device="cuda").expand(6, 5, 64)):
        _check_grad(embedding_backward(part, ids, 50), part, ids, 50, 1.0)
    none = torch.empty(0, 3, dtype=torch.int64, device="cuda")
    assert embedding_forward(none, wide).shape == (0, 3, 80)
    got = embedding_backward(torch.empty(0, 3, 80, device="cuda"), none, 50)
    assert got.shape == (50, 80) and not got.any()
    one = embedding_forward(torch.tensor(3, device="cuda"), wide)
    assert one.shape == (80,) and torch.equal(one, wide[3])


def test_rows_behind_a_padded_batch_and_nan():
    """A gradient that is not finite stays in its row; NaN in a padding token's place does not come through."""
    from haste_b200.embedding import embedding_backward
    ids = torch.tensor([0, 4, 0, 2, 4], device="cuda")
    dy = torch.ones(5, 32, device="cuda")
    dy[0], dy[2], dy[3] = float("nan"), float("inf"), float("inf")
    got = embedding_backward(dy, ids, 6, 1.0, 0)
    assert not got[[0, 1, 3, 5]].any() and got[2].isinf().all() and torch.equal(got[4], torch.full((32,), 2.0, device="cuda"))


def test_autograd_and_module():
    from haste_b200.embedding import Embedding, embedding
    torch.manual_seed(0)
    m, ref = Embedding(100, 48, padding_idx=3, scale=2.0, device="cuda"), torch.nn.Embedding(100, 48, padding_idx=3, device="cuda")
    ref.load_state_dict(m.state_dict())
    ids = torch.randint(0, 100, (7, 9), device="cuda")
    w = torch.randn(7, 9, 48, device="cuda")
    for y, times in ((m(ids), 1.0), (ref(ids), 2.0)):
        (y * w).sum().mul(times).backward()
    assert torch.equal(m(ids), 2 * ref(ids)) and torch.allclose(m.weight.grad, ref.weight.grad, rtol=0, atol=64 * 2 ** -24 * 2 * float(w.abs().max()) * 64)
    assert not m.weight.grad[3].any()
    with pytest.raises(RuntimeError):
        embedding(ids, m.weight, padding_idx=100)
    with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
        embedding(ids, torch.autograd.forward_ad.make_dual(m.weight.detach(), m.weight.detach()))
    y = embedding(ids, m.weight)
    g, = torch.autograd.grad(y.sum(), m.weight, create_graph=True)
    assert not g.requires_grad


def test_refusals():
    from haste_b200.embedding import embedding_backward, embedding_forward
    table, ids, dy = torch.randn(10, 8, device="cuda"), torch.tensor([1, 2], device="cuda"), torch.randn(2, 8, device="cuda")
    for call in (lambda: embedding_forward(ids.cpu(), table), lambda: embedding_forward(ids, table.cpu()), lambda: embedding_forward(ids.float(), table),
                 lambda: embedding_forward(ids, table.half()), lambda: embedding_forward(ids, table[0]), lambda: embedding_forward(ids, table[:0]),
                 lambda: embedding_backward(dy, ids[:1], 10), lambda: embedding_backward(dy, ids, 0), lambda: embedding_backward(dy.half(), ids, 10),
                 lambda: embedding_backward(dy, ids, 10, dtype=torch.float16), lambda: embedding_backward(dy, ids, 10, 1.0, 10), lambda: embedding_backward(dy, ids, 10, 1.0, -11),
                 lambda: embedding_backward(dy.cpu(), ids, 10), lambda: embedding_backward(dy, ids, 2 ** 31)):
        with pytest.raises(RuntimeError):
            call()


def test_in_a_graph_and_on_another_stream():
    from haste_b200.embedding import embedding_backward, embedding_forward
    table, ids, dy = torch.randn(500, 96, device="cuda"), torch.randint(0, 500, (3000,), device="cuda"), torch.randn(3000, 96, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = embedding_forward(ids, table), embedding_backward(dy, ids, 500)
    torch.cuda.synchronize()
    graphs, out = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out.append((embedding_forward(ids, table), embedding_backward(dy, ids, 500)))
        graphs.append(graph)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for pair in out:
        assert all(torch.equal(a, b) for a, b in zip(pair, want))
    ids.copy_(torch.randint(0, 500, (3000,), device="cuda"))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0][0], table[ids])
    _check_grad(out[0][1], dy, ids, 500, 1.0)

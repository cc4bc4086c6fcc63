"""Tensors that are views into flat buffers, off the boundaries that wide loads and stores want, with sizes that would allow them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF, F32 = torch.bfloat16, torch.float32


def _views(tensors, off):
    """The same tensors in one buffer, each `off` elements behind a multiple of 16."""
    at, places = 0, []
    for t in tensors:
        places.append(at + off)
        at += (t.numel() + off + 15) // 16 * 16
    flat = torch.zeros(at + 32, dtype=tensors[0].dtype, device="cuda")
    out = [flat[p:p + t.numel()].view(t.shape) for p, t in zip(places, tensors)]
    for o, t in zip(out, tensors):
        o.copy_(t)
    return flat, out


SHAPES = [(128, 192), (192, 128), (64, 64), (100, 36), (36, 100)]


@pytest.mark.parametrize("types", [(BF, BF), (F32, F32), (BF, F32), (F32, BF)])
@pytest.mark.parametrize("offs", [(1, 0), (0, 1), (2, 3), (3, 2), (8, 4)])
def test_muon(types, offs):
    from haste_b200.optim import moment_offsets, muon_step
    gen = torch.Generator().manual_seed(1)
    w, g = ([(0.02 * torch.randn(s, generator=gen)).to(t).cuda() for s in SHAPES] for t in types)
    at = moment_offsets([x.numel() for x in w])
    m = 1e-3 * torch.randn(at[-1], generator=gen).cuda()
    (flat, w2), (_, g2) = _views(w, offs[0]), _views(g, offs[1])
    used = torch.zeros(flat.numel(), dtype=torch.bool, device="cuda")
    for x in w2:
        used[x.storage_offset():x.storage_offset() + x.numel()] = True
    m2 = m.clone()
    for sr in (True, False):
        muon_step(w, g, m, step=2, lr=0.01, stochastic_rounding=sr)
        muon_step(w2, g2, m2, step=2, lr=0.01, stochastic_rounding=sr)
        assert all(torch.equal(a, b) for a, b in zip(w, w2)) and torch.equal(m, m2)
    assert not flat[~used].any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("off", [1, 2, 3, 4])
def test_orthogonalize(dtype, off):
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(2)
    g = [torch.randn(s, generator=gen).to(dtype).cuda() for s in SHAPES]
    assert all(torch.equal(a, b) for a, b in zip(orthogonalize(_views(g, off)[1]), orthogonalize(g)))


def test_momentum_off_its_boundary_is_refused():
    from haste_b200.optim import muon_step
    w, g = torch.zeros(16, 16, device="cuda"), torch.ones(16, 16, device="cuda")
    m = torch.zeros(300, device="cuda")
    with pytest.raises(RuntimeError, match="aligned"):
        muon_step([w], [g], m[1:257], step=1)
    assert not w.any() and not m.any()


@pytest.mark.parametrize("off", [1, 4, 7])
@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 32, 40, 300])
def test_gated_block(T, off):
    from haste_b200.feedforward import gated_backward, gated_forward
    D, F, O = 64, 136, 72
    gen = torch.Generator().manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=gen)
    aligned = [t.to(BF).cuda() for t in (r(F, D) * D ** -0.5, r(F, D) * D ** -0.5, r(O, F) * F ** -0.5, r(T, D), r(T, O))]
    want = gated_forward(aligned[3], *aligned[:3], keep=True)
    grads = gated_backward(aligned[4], aligned[3], *aligned[:3], *want[1:])
    exact, tol = eo.gated(aligned[3], *aligned[:3], "silu")
    for which in ((0,), (1,), (2,), (3,), (4,), (0, 1, 2, 3, 4)):
        ts = [_views([t], off)[1][0] if i in which else t for i, t in enumerate(aligned)]
        got = gated_forward(ts[3], *ts[:3], keep=True)
        for a, b, e in zip(got, exact, tol):
            assert eo.outside(a, b, e) is None
        if T > 32:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(gated_backward(ts[4], ts[3], *ts[:3], *want[1:]), grads))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("off", [1, 2, 4])
def test_embedding(dtype, off):
    from haste_b200.embedding import embedding_backward, embedding_forward
    gen = torch.Generator().manual_seed(off)
    table, dy, ids = torch.randn(50, 64, generator=gen).to(dtype).cuda(), torch.randn(300, 64, generator=gen).to(dtype).cuda(), torch.randint(0, 50, (300,), generator=gen).cuda()
    assert torch.equal(embedding_forward(ids, _views([table], off)[1][0], 1.5), embedding_forward(ids, table, 1.5))
    assert torch.equal(embedding_backward(_views([dy], off)[1][0], ids, 50, 1.5), embedding_backward(dy, ids, 50, 1.5))
    for kind in (torch.int64, torch.int32):
        near = _views([ids.to(kind)], off)[1][0]
        assert torch.equal(embedding_forward(near, table), embedding_forward(ids, table)) and torch.equal(embedding_backward(dy, near, 50), embedding_backward(dy, ids, 50))

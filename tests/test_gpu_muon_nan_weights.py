"""Weights that are NaN or infinite, or become so, in a Muon step: bf16 with stochastic rounding keeps them where the fp32 step has them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
# whole tiles of 64 x 64, rows that start off four elements, both orientations, one element
SHAPES = [(128, 192), (192, 128), (37, 21), (21, 37), (70, 66), (1, 1)]


def _inputs(seed):
    gen = torch.Generator().manual_seed(seed)
    g = [torch.randn(s, generator=gen).cuda() * 1e-3 for s in SHAPES]
    w = [(0.02 * torch.randn(s, generator=gen)).to(BF).cuda() for s in SHAPES]
    return g, w, torch.Generator().manual_seed(seed + 100)


def _steps(w, g, **kw):
    """The same step of fp32 weights, of bf16 ones rounded stochastically, and of bf16 ones rounded to nearest."""
    from haste_b200.optim import moment_offsets, muon_step
    out = []
    for weights, sr in (([x.float() for x in w], True), ([x.clone() for x in w], True), ([x.clone() for x in w], False)):
        muon_step(weights, g, torch.zeros(moment_offsets([x.numel() for x in w])[-1], device="cuda"), stochastic_rounding=sr, **kw)
        out.append(weights)
    return out


def _compare(exact, rounded, nearest):
    for e, r, n in zip(exact, rounded, nearest):
        assert torch.equal(r.isnan(), e.isnan()) and torch.equal(n.isnan(), e.isnan())
        inf = e.isinf()
        assert torch.equal(r[inf].float(), e[inf])
        fine = e.isfinite()
        # a whole step of bf16 (2^-7 of the value) at most, or of its smallest numbers
        assert ((r[fine].double() - e[fine].double()).abs() <= 2.0 ** -7 * e[fine].double().abs() + 2.0 ** -133).all()


@pytest.mark.parametrize("seed", range(4))
def test_weights_that_are_not_finite(seed):
    g, w, gen = _inputs(seed)
    for x in w:
        flat = x.view(-1)
        at = torch.randperm(flat.numel(), generator=gen)[:max(1, flat.numel() // 5)]
        values = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=BF)[torch.randint(0, 3, (len(at),), generator=gen)]
        if len(at) == 1:
            values[:] = float("nan")
        flat[at.cuda()] = values.cuda()
    before = [x.clone() for x in w]
    exact, rounded, nearest = _steps(w, g, step=3 + seed, lr=0.01, seed=seed)
    assert all(torch.equal(e.isnan(), x.isnan()) and torch.equal(e.isinf(), x.isinf()) for e, x in zip(exact, before))
    _compare(exact, rounded, nearest)


def test_steps_that_diverge():
    """Coefficients by which X leaves fp16: what becomes NaN in the fp32 step is NaN, not zero."""
    g, w, _ = _inputs(9)
    exact, rounded, nearest = _steps(w, g, step=1, lr=0.01, coefficients=(1e4, 0.0, 0.0))
    assert any(e.isnan().any() for e in exact)
    _compare(exact, rounded, nearest)

"""Matrices of few rows or columns in Newton-Schulz steps and the Muon update, element by element: a few roundings on the way do not average out there, so there are none to less than 32 bits."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do
from oracle import encoder_oracle as eo

BF, F32, U = torch.bfloat16, torch.float32, do.U


def _gradient(shape, gen, kind="low rank"):
    g = torch.randn(*shape, generator=gen)
    if kind == "low rank":
        few = max(1, min(shape) // 16)
        g = 5 * (torch.randn(shape[0], few, generator=gen) @ torch.randn(few, shape[1], generator=gen)) + g
    return g * 1e-3


def _check(got, g, what, **kw):
    """The result's own rounding to 32 bits and to bf16, and nothing that can be seen beside it."""
    want = eo.orthogonalize(g, **kw)
    bad = eo.outside(got, want, U * want.abs() + 1e-11, what)
    assert got.dtype == BF and bad is None, bad


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", range(1, 33))
def test_every_number_of_rows(rows, dtype):
    from haste_b200.optim import orthogonalize
    gen, rng = torch.Generator().manual_seed(rows), random.Random(rows)
    shapes = [(rows, max(rows, q)) for q in (1, 2, 3, 5, 31, 32, 33, 63, 64, 65, 127, 200, 256, 511, 512, 513, 1030)] + [(rows, rng.randint(rows, 3000)) for _ in range(3)]
    g = [_gradient(s, gen, kind).to(dtype).cuda() for s in shapes for kind in ("low rank", "gauss")]
    g += [x.t().contiguous() for x in g]
    got = orthogonalize(g)
    for a, b in zip(got, g):
        _check(a, b, f"{tuple(b.shape)}")
    assert all(torch.equal(a, b) for a, b in zip(got, orthogonalize(g)))
    for i in (0, len(g) // 2, len(g) - 1):
        assert torch.equal(orthogonalize([g[i]])[0], got[i])                     # whatever stands beside it


@pytest.mark.parametrize("shape", [(2, 3), (2, 9), (2, 300), (1, 3), (3, 40), (4, 4)])
def test_many_draws(shape):
    """Hundreds of matrices of the sizes at which roundings of products to 16 bits show most, in one call."""
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(shape[1])
    g = [_gradient(shape, gen).cuda() for _ in range(400)]
    for a, b in zip(orthogonalize(g), g):
        _check(a, b, f"{shape}")


@pytest.mark.parametrize("shape", [(1, 100000), (100000, 1), (7, 40001), (40001, 7), (32, 70000), (20, 300000), (300000, 20)])
def test_long_ones(shape):
    from haste_b200.optim import orthogonalize
    g = _gradient(shape, torch.Generator().manual_seed(shape[0])).cuda()
    _check(orthogonalize([g])[0], g, f"{shape}")


def test_steps_coefficients_and_scales():
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(3)
    for shape in ((3, 70), (31, 31), (32, 17)):
        g = _gradient(shape, gen).cuda()
        for steps in (1, 2, 6, 9):
            _check(orthogonalize([g], steps)[0], g, f"{steps} steps", steps=steps)
        _check(orthogonalize([g], 12, (1.5, -0.5, 0.0))[0], g, "another polynomial", steps=12, coefficients=(1.5, -0.5, 0.0))
        for scale in (1e-3, 1e18, 1e38):
            _check(orthogonalize([g * scale])[0], g * scale, f"times {scale}")
        _check(orthogonalize([g * 1e-30], eps=2.0 ** -100)[0], g * 1e-30, "tiny", eps=2.0 ** -100)
        _check(orthogonalize([g * 1e-10])[0], g * 1e-10, "below eps")
        assert not orthogonalize([torch.zeros_like(g)])[0].any()
        for bad in (float("nan"), float("inf")):
            h = g.clone()
            h[2, 1] = bad
            out = orthogonalize([g, h, g.t().contiguous()])
            assert out[1].isnan().all() and torch.equal(out[0], orthogonalize([g])[0]) and out[2].isfinite().all()


@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw"])
@pytest.mark.parametrize("types", [(BF, BF), (F32, F32), (BF, F32), (F32, BF)])
def test_step(types, adjust):
    from haste_b200.optim import moment_offsets, muon_step
    gen = torch.Generator().manual_seed(4)
    shapes = [(1, 1), (5, 300), (300, 5), (31, 33), (33, 31), (32, 32), (2, 3), (17, 600), (600, 18), (40, 50), (1, 999), (64, 3)]
    at = moment_offsets([a * b for a, b in shapes])
    w = [(0.02 * torch.randn(s, generator=gen)).to(types[0]).cuda() for s in shapes]
    g = [_gradient(s, gen).to(types[1]).cuda() for s in shapes]
    m = torch.full((at[-1],), 7.0, device="cuda")
    for a, s in zip(at, shapes):
        m[a:a + s[0] * s[1]] = _gradient(s, gen).cuda().view(-1)
    g[3] = None
    g[6][1, 1] = float("nan")
    old_w, old_m = [x.clone() for x in w], m.clone()
    lr, mu, decay = 0.02, 0.9, 0.1
    muon_step(w, g, m, step=7, lr=lr, momentum=mu, nesterov=False, weight_decay=decay, adjust=adjust, stochastic_rounding=False)
    for i, s in enumerate(shapes):
        part = slice(at[i], at[i] + s[0] * s[1])
        new = m[part].double().view(s)
        if i in (3, 6):
            assert torch.equal(w[i], old_w[i]) and torch.equal(m[part], old_m[part])
            continue
        before = old_m[part].double().view(s)
        assert do.outside(m[part].view(s), mu * before + (1 - mu) * g[i].double(), 3 * U * (before.abs() + g[i].double().abs()), "m") is None
        if min(s) > 32:
            continue
        # without Nesterov's form what is made orthogonal is the momentum as it is stored; rate, decay, X, a product and the sum are rounded to 32 bits
        x, rate = eo.orthogonalize(new), eo.muon_rate(s, lr, adjust)
        want = old_w[i].double() * (1 - lr * decay) - rate * x
        assert eo.outside(w[i], want, 4 * U * (old_w[i].double().abs() + rate * x.abs()), f"w {s}") is None
    used = torch.zeros_like(m, dtype=torch.bool)
    for a, s in zip(at, shapes):
        used[a:a + s[0] * s[1]] = True
    assert (m[~used] == 7).all()


def test_nesterov_and_random_bits():
    """The direction of Nesterov's form, and stochastic rounding of what fp32 weights become, at every place of four neighbours."""
    import numpy as np
    from haste_b200.optim import moment_offsets, muon_step
    from oracle.philox import philox4x32
    gen = torch.Generator().manual_seed(5)
    shapes = [(37, 21), (21, 37), (3, 10), (64, 8), (8, 64), (1, 5)]
    at = moment_offsets([a * b for a, b in shapes])
    g = [_gradient(s, gen).cuda() for s in shapes]
    w = [(0.02 * torch.randn(s, generator=gen)).to(BF).cuda() for s in shapes]
    old = [x.clone() for x in w]
    m = torch.zeros(at[-1], device="cuda")
    m0 = [_gradient(s, gen).cuda() for s in shapes]
    for a, x in zip(at, m0):
        m[a:a + x.numel()] = x.view(-1)
    args = dict(step=5, lr=0.01, momentum=0.9, weight_decay=0.1, seed=77, stream_index=3)
    exact = [x.float() for x in w]
    muon_step(exact, g, m.clone(), **args)
    muon_step(w, g, m, **args)
    for i, s in enumerate(shapes):
        n, first = s[0] * s[1], at[i]
        u = 0.9 * (0.9 * m0[i].double() + 0.1 * g[i].double()) + 0.1 * g[i].double()
        rate = eo.muon_rate(s, 0.01, "original")
        want = old[i].double() * (1 - 0.01 * 0.1) - rate * eo.orthogonalize(u)
        # u is rounded to 32 bits, and five steps multiply that by 3.4445^5 = 485 at most
        assert float((exact[i].double() - want).norm()) <= 2 * 485 * U * rate * min(s) ** 0.5 + 4 * U * float(want.norm() + old[i].double().norm()), s
        c = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
        words = np.stack(philox4x32(c & np.uint64(0xFFFFFFFF), c >> np.uint64(32), 3, 2, 77, 5, rounds=7), 1).reshape(-1)[first % 4:first % 4 + n]
        r = torch.from_numpy((words & 0xFFFF).astype(np.int64)).cuda().int().view(s)
        assert torch.equal(w[i].view(torch.int16), ((exact[i].view(torch.int32) + r) >> 16).to(torch.int16))


def test_more_than_a_launch_holds():
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(6)
    shapes = [(1 + i % 32, 1 + i * 7 % 211) for i in range(500)] + [(100, 200), (64, 64)]
    g = [_gradient(s, gen).cuda() for s in shapes]
    for a, b in zip(orthogonalize(g), g):
        if min(b.shape) <= 32:
            _check(a, b, f"{tuple(b.shape)}")
        else:
            want, tol = eo.orthogonalize_bound(b)
            assert float((a.double() - want).norm()) <= tol


def test_in_graphs():
    from haste_b200.optim import moment_offsets, muon_step, orthogonalize
    gen = torch.Generator().manual_seed(7)
    g = [_gradient(s, gen).cuda() for s in ((3, 400), (400, 30), (100, 64))]
    want = orthogonalize(g)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(orthogonalize(g))
        graphs.append(graph)
    w, m = [torch.zeros_like(x) for x in g], torch.zeros(moment_offsets([x.numel() for x in g])[-1], device="cuda")
    w2, m2 = [x.clone() for x in w], m.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(w, g, m, step=1)
    for _ in range(2):
        for h in (*graphs, graph):
            h.replay()
        muon_step(w2, g, m2, step=1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(w, w2)) and torch.equal(m, m2)

"""Newton-Schulz steps and the Muon update against the 64-bit oracle: shapes, types, what a step leaves alone, random bits, the optimizer's state."""
import copy
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do
from oracle import encoder_oracle as eo
from oracle.philox import philox4x32

BF, F32 = torch.bfloat16, torch.float32
SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 5), (16, 16), (31, 33), (33, 31), (64, 64), (64, 200), (255, 257), (256, 256), (257, 255), (300, 40), (40, 300), (512, 512), (384, 1000), (1000, 384),
          (769, 770)]


def _gradient(shape, kind, gen):
    g = torch.randn(*shape, generator=gen)
    if kind == "low rank":
        few = max(1, min(shape) // 16)
        g = torch.randn(shape[0], few, generator=gen) @ torch.randn(few, shape[1], generator=gen) + 0.05 * g
    return g * 1e-3


def _check(got, g, steps=5, coefficients=(eo.A, eo.B, eo.C), eps=1e-7, what=""):
    want, tol = eo.orthogonalize_bound(g, steps, coefficients, eps)
    assert got.dtype == BF and got.shape == want.shape
    off = float((got.double() - want).norm())
    assert off <= tol, f"{what}: off by {off:.3g}, {tol:.3g} allowed, of {float(want.norm()):.3g}"


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["gauss", "low rank"])
def test_orthogonalize(kind, dtype):
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(3)
    g = [_gradient(s, kind, gen).to(dtype).cuda() for s in SHAPES]
    got = orthogonalize(g)
    for a, b in zip(got, g):
        _check(a, b, what=f"{tuple(b.shape)}")
    assert all(torch.equal(a, b) for a, b in zip(got, orthogonalize(g)))
    alone = orthogonalize([g[5]])[0]
    assert torch.equal(alone, got[5])                                           # whatever stands beside it


def test_steps_and_coefficients():
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(4)
    g = _gradient((130, 200), "gauss", gen).cuda()
    for steps in (1, 2, 3, 6):
        _check(orthogonalize([g], steps)[0], g, steps)
    _check(orthogonalize([g], 8, (1.5, -0.5, 0.0))[0], g, 8, (1.5, -0.5, 0.0))
    s = torch.linalg.svdvals(orthogonalize([g])[0].float())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


def test_many_of_one_shape_and_many_shapes():
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(5)
    shapes = [(96, 96)] * 30 + [(8 * i + 1, 50) for i in range(1, 40)] + [(50, 96), (96, 50)] * 3 + [(20 + i % 3, 30) for i in range(150)]
    g = [_gradient(s, "gauss", gen).cuda() for s in shapes]
    for a, b in zip(orthogonalize(g), g):
        _check(a, b, what=f"{tuple(b.shape)}")


def test_more_shapes_and_matrices_than_a_launch_holds():
    """Shapes that differ by their multiples of 64 in each direction, more of them than one launch's parameters, in the wide form and in the narrow one; matrices that fill two
    groups, and a round of the workspace."""
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(51)
    shapes = [(64 * i + 1, 64 * j + 3) for i in range(7) for j in range(i, 7)]
    g = [_gradient(s, "gauss", gen).cuda() for s in shapes]
    for a, b in zip(orthogonalize(g), g):
        _check(a, b, what=f"{tuple(b.shape)}")
    g = [_gradient(s, "gauss", gen).cuda() for s in shapes] * 6
    got = orthogonalize(g)
    for i in (0, 27, 28, 100, 167):
        _check(got[i], g[i], what=f"{tuple(g[i].shape)}")
        assert torch.equal(got[i], got[i % 28])
    one = [_gradient((1024, 1024), "gauss", gen).cuda() for _ in range(3)]
    for count in (48, 150):
        got = orthogonalize([one[i % 3] for i in range(count)])
        for i in range(3):
            _check(got[i], one[i])
        assert all(torch.equal(x, got[i % 3]) for i, x in enumerate(got))


def test_scales_zeros_and_what_is_not_finite():
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(6)
    g = _gradient((60, 90), "gauss", gen).cuda()
    for scale in (1e-3, 1e18, 1e33):
        _check(orthogonalize([g * scale])[0], g * scale)
    tiny = g * 1e-30
    _check(orthogonalize([tiny], 5, (eo.A, eo.B, eo.C), 2.0 ** -100)[0], tiny, eps=2.0 ** -100)
    bad, worse = g.clone(), g.t().contiguous()
    bad[3, 4], worse[5, 6] = float("nan"), float("inf")
    out = orthogonalize([g, torch.zeros_like(g), bad, worse, g[:0]])
    _check(out[0], g)
    assert not out[1].any() and out[2].isnan().all() and out[3].isnan().all() and out[4].shape == (0, 90)
    assert orthogonalize([]) == []


def test_large_and_long():
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(7)
    for shape in ((2048, 1024), (30, 40000), (1536, 1536)):
        g = _gradient(shape, "low rank", gen).cuda()
        _check(orthogonalize([g])[0], g, what=f"{shape}")


def _words(first, n, seed, step, stream):
    i = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    return np.stack(philox4x32(i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), stream, 2, seed, step, rounds=7), 1).reshape(-1)[first % 4:first % 4 + n]


@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw"])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("types", [(BF, BF), (F32, F32), (BF, F32), (F32, BF)])
def test_step(types, nesterov, adjust):
    from haste_b200.optim import moment_offsets, muon_step
    gen = torch.Generator().manual_seed(8)
    shapes = [(70, 33), (16, 16), (5, 300), (33, 70), (129, 64), (1, 1)]
    at = moment_offsets([a * b for a, b in shapes])
    w = [(0.02 * torch.randn(s, generator=gen)).to(types[0]).cuda() for s in shapes]
    g = [_gradient(s, "gauss", gen).to(types[1]).cuda() for s in shapes]
    m = torch.zeros(at[-1], device="cuda")
    for a, s in zip(at, shapes):
        m[a:a + s[0] * s[1]] = _gradient(s, "gauss", gen).cuda().view(-1)
    g[3] = None
    old_w, old_m = [x.clone() for x in w], m.clone()
    lr, mu, decay = 0.02, 0.9, 0.1
    muon_step(w, g, m, step=7, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, adjust=adjust, stochastic_rounding=False)
    for i, s in enumerate(shapes):
        n = s[0] * s[1]
        before = old_m[at[i]:at[i] + n].double().view(s)
        if g[i] is None:
            assert torch.equal(w[i], old_w[i]) and torch.equal(m[at[i]:at[i] + n].view(s).double(), before)
            continue
        new = mu * before + (1 - mu) * g[i].double()
        tol = 3 * do.U * (before.abs() + g[i].double().abs())
        assert do.outside(m[at[i]:at[i] + n].view(s), new, tol, "m") is None
        u = mu * new + (1 - mu) * g[i].double() if nesterov else new
        x, tol_x = eo.orthogonalize_bound(u)
        rate = eo.muon_rate(s, lr, adjust)
        want = old_w[i].double() * (1 - lr * decay) - rate * x
        # the direction's error, and half a step of the weights' type for each of them
        off = float((w[i].double() - want).norm())
        assert off <= rate * tol_x + (do.HALF_ULP[types[0]] + 3 * do.U) * float(want.norm()), (s, off)
    used = torch.zeros_like(m, dtype=torch.bool)
    for a, s in zip(at, shapes):
        used[a:a + s[0] * s[1]] = True
    assert torch.equal(m[~used], old_m[~used])


def test_random_bits():
    from haste_b200.optim import moment_offsets, muon_step
    gen = torch.Generator().manual_seed(9)
    shapes = [(37, 21), (64, 128), (50, 13)]
    at = moment_offsets([a * b for a, b in shapes])
    g = [_gradient(s, "gauss", gen).cuda() for s in shapes]
    w = [(0.02 * torch.randn(s, generator=gen)).to(BF).cuda() for s in shapes]
    args = dict(step=5, lr=0.01, weight_decay=0.1, seed=77, stream_index=3)
    exact = [x.float() for x in w]
    muon_step(exact, g, torch.zeros(at[-1], device="cuda"), **args)             # the same weights in fp32
    muon_step(w, g, torch.zeros(at[-1], device="cuda"), **args)
    for i, s in enumerate(shapes):
        n = s[0] * s[1]
        r = torch.from_numpy((_words(at[i], n, 77, 5, 3) & 0xFFFF).astype(np.int64)).cuda().int().view(s)
        want = ((exact[i].view(torch.int32) + r) >> 16).to(torch.int16).view(BF)
        assert torch.equal(w[i].view(torch.int16), want.view(torch.int16))


def test_what_is_not_finite_changes_nothing():
    from haste_b200.optim import moment_offsets, muon_step
    gen = torch.Generator().manual_seed(10)
    shapes = [(20, 30), (30, 20), (20, 20)]
    at = moment_offsets([a * b for a, b in shapes])
    for bad in (float("nan"), float("inf"), -float("inf")):
        w, g = [torch.randn(s, generator=gen).to(BF).cuda() for s in shapes], [_gradient(s, "gauss", gen).cuda() for s in shapes]
        g[1][2, 3] = bad
        m = torch.rand(at[-1], device="cuda") * 1e-3
        old, old_m = [x.clone() for x in w], m.clone()
        muon_step(w, g, m, step=1)
        assert torch.equal(w[1], old[1]) and torch.equal(m[at[1]:at[2]], old_m[at[1]:at[2]])
        assert not torch.equal(w[0], old[0]) and not torch.equal(w[2], old[2]) and not torch.equal(m[:600], old_m[:600])


def test_refusals():
    from haste_b200.optim import Muon, muon_step, orthogonalize
    a, b, m = torch.randn(4, 6, device="cuda"), torch.randn(4, 6, device="cuda"), torch.zeros(256, device="cuda")
    for call in (lambda: orthogonalize([a.cpu()]), lambda: orthogonalize([a.view(-1)]), lambda: orthogonalize([a.half()]), lambda: orthogonalize([a.t()]), lambda: orthogonalize([a, a.to(BF)]),
                 lambda: orthogonalize([a, None]), lambda: orthogonalize([a], 0), lambda: orthogonalize([a], eps=0.0), lambda: orthogonalize([a], 5, (float("nan"), 0.0, 0.0)),
                 lambda: muon_step([a], [b, b], m, step=1), lambda: muon_step([a], [b[:2]], m, step=1), lambda: muon_step([a], [b], m[:100], step=1), lambda: muon_step([a], [b], m.cpu(), step=1),
                 lambda: muon_step([a], [b], m, step=0), lambda: muon_step([a], [b], m, step=1, lr=-1.0), lambda: muon_step([a], [b], m, step=1, momentum=1.0),
                 lambda: muon_step([a], [b], m, step=1, adjust="rms"), lambda: muon_step([a, a], [b, b], torch.zeros(512, device="cuda"), step=1), lambda: muon_step([a.view(-1)], [b.view(-1)], m, step=1), lambda: muon_step([a], [b], m.to(BF), step=1)):
        with pytest.raises(RuntimeError):
            call()
    muon_step([a], [None], m, step=1)
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(adjust="rms"), dict(steps=0), dict(weight_decay=-0.1), dict(eps=0.0)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(a)], **kw)
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(a.view(-1))])


def _model(dtype):
    torch.manual_seed(11)
    return [torch.nn.Parameter(torch.randn(s, device="cuda").to(dtype) * 0.02) for s in ((40, 60), (60, 40), (32, 32))]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_optimizer_is_the_function(dtype):
    from haste_b200.optim import Muon, moment_offsets, muon_step
    params = _model(dtype)
    mine = [p.detach().clone() for p in params]
    opt = Muon(params, lr=0.01, weight_decay=0.05, adjust="match_rms_adamw", seed=5)
    m = torch.zeros(moment_offsets([p.numel() for p in params])[-1], device="cuda")
    for t in range(1, 4):
        grads = [torch.randn(p.shape, device="cuda").to(dtype) * 1e-3 if (i + t) % 3 else None for i, p in enumerate(params)]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        muon_step(mine, grads, m, step=t, lr=0.01, weight_decay=0.05, adjust="match_rms_adamw", seed=5)
        assert all(torch.equal(a, b) for a, b in zip(params, mine))
    assert set(opt.state[params[0]]) == {"momentum_buffer"} and opt.state[params[0]]["momentum_buffer"].shape == params[0].shape


def test_state_goes_on():
    from haste_b200.optim import Muon
    params = _model(BF)
    opt = Muon(params, lr=0.01)
    grads = [[torch.randn(p.shape, device="cuda").to(BF) * 1e-3 for p in params] for _ in range(4)]

    def steps(ps, o, some):
        for gs in some:
            for p, g in zip(ps, gs):
                p.grad = g
            o.step()

    steps(params, opt, grads[:2])
    saved, weights = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in params]
    steps(params, opt, grads[2:])
    again = [torch.nn.Parameter(w) for w in weights]
    other = Muon(again, lr=0.5)
    other.load_state_dict(saved)
    steps(again, other, grads[2:])
    assert all(torch.equal(a, b) for a, b in zip(params, again))
    third = copy.deepcopy(other)
    assert third.param_groups[0]["step_count"] == 4 and all(torch.equal(third.state[p]["momentum_buffer"], opt.state[q]["momentum_buffer"]) for p, q in zip(third.param_groups[0]["params"], params))


def test_state_of_torchs_class():
    from haste_b200.optim import Muon
    if not hasattr(torch.optim, "Muon"):
        pytest.skip("this torch has no Muon")
    params = _model(BF)
    theirs = torch.optim.Muon(params, lr=0.01)
    for p in params:
        p.grad = torch.randn(p.shape, device="cuda").to(BF) * 1e-3
    theirs.step()
    opt = Muon(params, lr=0.5)
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 0.01
    for p in params:
        p.grad = torch.randn(p.shape, device="cuda").to(BF) * 1e-3
    want = {p: 0.95 * theirs.state[p]["momentum_buffer"].double() + 0.05 * p.grad.double() for p in params}
    opt.step()
    for p in params:
        assert do.outside(opt.state[p]["momentum_buffer"], want[p], 3 * do.U * 2 * want[p].abs().amax().expand(p.shape), "m") is None


def test_in_a_graph():
    from haste_b200.optim import muon_step, orthogonalize
    gen = torch.Generator().manual_seed(12)
    g = [_gradient(s, "gauss", gen).cuda() for s in ((100, 64), (64, 100), (30, 30))]
    want = orthogonalize(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        orthogonalize(g)
    torch.cuda.synchronize()
    outs, graphs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(orthogonalize(g))
        graphs.append(graph)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))
    w, m = [torch.zeros_like(x) for x in g], torch.zeros(256 * 60, device="cuda")
    version = w[0]._version
    muon_step(w, g, m, step=1)
    assert w[0]._version > version and m._version > 0


def test_rounds_of_a_list_with_gaps():
    """Matrices of more scratch memory than one round takes: without one of them the others stay in the rounds that the whole list's memory was asked for."""
    from haste_b200 import _lib
    from haste_b200.optim import moment_offsets, muon_step
    shapes = [(64, 1677696), (64, 1258304), (64, 1090496)]
    sizes = lambda which: ((ctypes.c_int64 * len(which))(*(shapes[i][0] for i in which)), (ctypes.c_int64 * len(which))(*(shapes[i][1] for i in which)), len(which))
    assert _lib.lib.haste_muon_scratch(*sizes([0, 2])) > _lib.lib.haste_muon_scratch(*sizes([0, 1, 2])) > _lib.lib.haste_muon_scratch(*sizes([0]))
    gen = torch.Generator(device="cuda").manual_seed(3)
    params = [torch.randn(s, generator=gen, device="cuda").to(BF) for s in shapes]
    grads = [torch.randn(s, generator=gen, device="cuda").to(BF) for s in shapes]
    alone = []
    for i in (0, 2):
        p = params[i].clone()
        muon_step([p], [grads[i]], torch.zeros(p.numel(), device="cuda"), step=1, lr=0.1, stochastic_rounding=False)
        alone.append(p)
    before = params[1].clone()
    muon_step(params, [grads[0], None, grads[2]], torch.zeros(moment_offsets([p.numel() for p in params])[-1], device="cuda"), step=1, lr=0.1, stochastic_rounding=False)
    assert torch.equal(params[0], alone[0]) and torch.equal(params[1], before) and torch.equal(params[2], alone[1])


def test_a_type_that_is_refused_changes_nothing():
    from haste_b200.optim import Muon
    fine, other = (torch.nn.Parameter(torch.ones(8, 8, device="cuda", dtype=t)) for t in (BF, torch.float16))
    opt = Muon([dict(params=[fine]), dict(params=[other])], lr=0.1)
    fine.grad, other.grad = torch.randn_like(fine), torch.randn_like(other)
    with pytest.raises(RuntimeError, match="float16"):
        opt.step()
    assert (fine == 1).all() and opt.param_groups[0]["step_count"] == 0
    other.grad = None
    opt.step()
    assert not (fine == 1).all()

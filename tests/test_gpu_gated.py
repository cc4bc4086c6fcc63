"""The gated feed-forward block against the 64-bit oracle: every activation, one row to thousands, odd sizes and strides, which gradients are wanted, autograd and differences."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF = torch.bfloat16
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]
# rows, D, F, O
SHAPES = [(1, 768, 2048, 768), (2, 16, 24, 8), (8, 64, 128, 64), (5, 77, 130, 33), (9, 64, 128, 64), (16, 8, 8, 8), (1, 1, 1, 1), (17, 1, 3, 2), (64, 768, 1024, 768), (100, 509, 1021, 509),
          (257, 72, 136, 264), (300, 512, 640, 512), (333, 1000, 257, 40), (128, 128, 2560, 128)]


def _inputs(T, D, F, O, seed=0, grow=1.0):
    gen = torch.Generator().manual_seed(seed * 101 + T * 7 + D * 3 + F)
    r = lambda *s: torch.randn(*s, generator=gen)
    x, wg, wu, wd, dy = r(T, D) * grow, r(F, D) * D ** -0.5, r(F, D) * D ** -0.5, r(O, F) * F ** -0.5, r(T, O) * 0.1
    return [t.to(BF).cuda() for t in (x, wg, wu, wd, dy)]


def _check(names, got, want, tol):
    for name, g, v, t in zip(names, got, want, tol):
        assert g.dtype == BF and g.shape == v.shape, name
        bad = eo.outside(g, v, t, name)
        assert bad is None, bad


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, act):
    from haste_b200.feedforward import gated_forward
    x, wg, wu, wd, _ = _inputs(*shape)
    got = gated_forward(x, wg, wu, wd, act, keep=True)
    _check(("y", "gate", "up"), got, *eo.gated(x, wg, wu, wd, act))
    y = gated_forward(x, wg, wu, wd, act)
    assert torch.equal(y, got[0])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, act):
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(*shape)
    _, gate, up = gated_forward(x, wg, wu, wd, act, keep=True)
    got = gated_backward(dy, x, wg, wu, wd, gate, up, act)
    _check(("dx", "dw_gate", "dw_up", "dw_down"), got, *eo.gated_grad(dy, x, wg, wu, wd, gate, up, act))
    assert all(torch.equal(a, b) for a, b in zip(got, gated_backward(dy, x, wg, wu, wd, gate, up, act)))


@pytest.mark.parametrize("T", [1, 8, 9, 127, 128, 129, 255, 256, 257, 511])
def test_rows_around_a_tile(T):
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(T, 200, 264, 136)
    got = gated_forward(x, wg, wu, wd, "silu", keep=True)
    _check(("y", "gate", "up"), got, *eo.gated(x, wg, wu, wd, "silu"))
    _check("x g u d".split(), gated_backward(dy, x, wg, wu, wd, *got[1:], "silu"), *eo.gated_grad(dy, x, wg, wu, wd, *got[1:], "silu"))


@pytest.mark.parametrize("shape", [(20000, 256, 512, 256), (5000, 320, 2048, 1024), (2049, 2048, 320, 64)])
def test_many_rows(shape):
    """Several tiles for every pair of SMs, weight gradients of long sums cut into parts."""
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(*shape)
    got = gated_forward(x, wg, wu, wd, "silu", keep=True)
    _check(("y", "gate", "up"), got, *eo.gated(x, wg, wu, wd, "silu"))
    grads = gated_backward(dy, x, wg, wu, wd, *got[1:], "silu")
    _check("x g u d".split(), grads, *eo.gated_grad(dy, x, wg, wu, wd, *got[1:], "silu"))


@pytest.mark.parametrize("act", ACTS)
def test_large_and_unusual_values(act):
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(40, 64, 72, 64, grow=30.0)
    got = gated_forward(x, wg, wu, wd, act, keep=True)
    _check(("y", "gate", "up"), got, *eo.gated(x, wg, wu, wd, act))
    _check("x g u d".split(), gated_backward(dy, x, wg, wu, wd, *got[1:], act), *eo.gated_grad(dy, x, wg, wu, wd, *got[1:], act))
    x[3, 5], x[7, 1] = float("nan"), float("inf")                          # stay in their rows
    for rows in (slice(0, 40), slice(0, 8)):
        y = gated_forward(x[rows], wg, wu, wd, act)
        assert y[3].isnan().all() and y[7].isnan().any() and y[[0, 1, 2, 4, 5, 6]].isfinite().all()
    big = torch.full((16, 64), -1e4, dtype=BF, device="cuda")              # gates far below zero
    y, g, u = gated_forward(big, wg.abs(), wu, wd, act, keep=True)
    assert not y.any() and all(t.isfinite().all() for t in gated_backward(dy[:16], big, wg.abs(), wu, wd, g, u, act))


def test_which_gradients():
    from haste_b200.feedforward import gated_backward, gated_forward
    for shape in ((40, 64, 72, 80), (40, 61, 73, 35)):
        x, wg, wu, wd, dy = _inputs(*shape)
        _, gate, up = gated_forward(x, wg, wu, wd, "silu", keep=True)
        every = gated_backward(dy, x, wg, wu, wd, gate, up)
        for bits in range(16):
            want = [bool(bits >> i & 1) for i in range(4)]
            got = gated_backward(dy, x, wg, wu, wd, gate, up, "silu", want)
            for w, g, e in zip(want, got, every):
                assert (g is None) == (not w) and (g is None or torch.equal(g, e))


def test_strides_shapes_and_no_rows():
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(60, 96, 40, 56)
    want = gated_forward(x, wg, wu, wd, keep=True)
    grads = gated_backward(dy, x, wg, wu, wd, *want[1:])
    wide = torch.zeros(60, 131, dtype=BF, device="cuda")
    for at in (0, 8, 3):
        wide[:, at:at + 96] = x
        got = gated_forward(wide[:, at:at + 96], wg, wu, wd, keep=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = x.t().contiguous().t()
    assert torch.equal(gated_forward(turned, wg, wu, wd), want[0])
    got = gated_forward(x.view(3, 4, 5, 96), wg, wu, wd, keep=True)
    assert got[0].shape == (3, 4, 5, 56) and got[1].shape == (3, 4, 5, 40) and torch.equal(got[0].view(60, 56), want[0])
    wide = torch.zeros(60, 77, dtype=BF, device="cuda")
    wide[:, 9:65], pad = dy, torch.zeros(60, 48, dtype=BF, device="cuda")
    pad[:, :40] = want[1]
    for args in ((wide[:, 9:65], x, wg, wu, wd, *want[1:]), (dy.view(6, 10, 56), x.view(6, 10, 96), wg, wu, wd, want[1].view(6, 10, 40), want[2].view(6, 10, 40)),
                 (dy, turned, wg, wu, wd, pad[:, :40], want[2])):
        got = gated_backward(*args)
        assert got[0].shape == args[1].shape and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, grads))
    one = torch.randn(56, device="cuda").to(BF)
    assert all(torch.equal(a, b) for a, b in zip(gated_backward(one.expand(60, 56), x, wg, wu, wd, *want[1:]), gated_backward(one.repeat(60, 1), x, wg, wu, wd, *want[1:])))
    y, g, u = gated_forward(x[:0], wg, wu, wd, keep=True)
    assert y.shape == (0, 56) and g.shape == (0, 40)
    got = gated_backward(dy[:0], x[:0], wg, wu, wd, g, u)
    assert got[0].shape == (0, 96) and not any(t.any() for t in got[1:])
    y = gated_forward(x[0], wg, wu, wd)
    assert y.shape == (56,)


def test_one_row_of_many():
    """A row's result in a large batch is that of the row alone, to the rounding of h."""
    from haste_b200.feedforward import gated_forward
    x, wg, wu, wd, _ = _inputs(600, 256, 512, 128)
    y = gated_forward(x, wg, wu, wd)
    for r in (0, 1, 255, 256, 599):
        (want, *_), (tol, *_) = eo.gated(x[r:r + 1], wg, wu, wd, "silu")
        assert eo.outside(gated_forward(x[r:r + 1], wg, wu, wd), want, tol) is None
    (want, *_), (tol, *_) = eo.gated(x, wg, wu, wd, "silu")
    assert eo.outside(y, want, tol) is None


def test_autograd_module_and_differences():
    from haste_b200.feedforward import GatedFeedForward, gated_feed_forward
    torch.manual_seed(1)
    for act in ACTS[:3]:
        m = GatedFeedForward(48, 80, out=32, activation=act, device="cuda")
        x = torch.randn(4, 5, 48, device="cuda").to(BF).requires_grad_()
        w = torch.randn(4, 5, 32, device="cuda")
        y = m(x)
        (y.float() * w).sum().backward()
        # the formula in 64 bits and its differences along a random direction
        params = [x, m.w_gate, m.w_up, m.w_down]

        def value(ts):
            (v, *_), _ = eo.gated(ts[0].reshape(20, 48), *ts[1:], act, few=1 << 30)
            return float((v * w.double().view(20, 32)).sum())

        for i, p in enumerate(params):
            d = torch.randn(p.shape, device="cuda", dtype=torch.float64)
            plus = [t.detach().double() + (1e-4 * d if i == j else 0) for j, t in enumerate(params)]
            minus = [t.detach().double() - (1e-4 * d if i == j else 0) for j, t in enumerate(params)]
            slope = (value(plus) - value(minus)) / 2e-4
            # the rounding of the incoming gradient, of dgate, dup or h, of the kept projections and of the result: 2^-8 each on every term
            assert abs(float((p.grad.double() * d).sum()) - slope) <= 6 * 2 ** -8 * float((p.grad.double() * d).abs().sum())
        with torch.no_grad():
            assert torch.equal(m(x), y)
    frozen = gated_feed_forward(x.detach(), m.w_gate.detach(), m.w_up.detach(), m.w_down, act)
    g, = torch.autograd.grad(frozen.float().sum(), m.w_down)
    assert g.shape == m.w_down.shape
    with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
        gated_feed_forward(x.detach(), m.w_gate.detach(), m.w_up.detach(), torch.autograd.forward_ad.make_dual(m.w_down.detach(), m.w_down.detach()), act)


def test_refusals():
    from haste_b200.feedforward import GatedFeedForward, gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(20, 16, 24, 8)
    _, gate, up = gated_forward(x, wg, wu, wd, keep=True)
    for call in (lambda: gated_forward(x.cpu(), wg, wu, wd), lambda: gated_forward(x.float(), wg, wu, wd), lambda: gated_forward(x, wg.float(), wu, wd), lambda: gated_forward(x, wg.cpu(), wu, wd),
                 lambda: gated_forward(x, wg[:, :8], wu, wd), lambda: gated_forward(x, wg, wu[:8], wd), lambda: gated_forward(x, wg, wu, wd[:, :8].contiguous()),
                 lambda: gated_forward(x, wg.t().contiguous().t(), wu, wd), lambda: gated_forward(x, wg, wu, wd, "tanh"), lambda: gated_forward(x[:, :0], wg, wu, wd),
                 lambda: gated_forward(x, wg, wu, wd[:0]), lambda: gated_backward(dy[:10], x, wg, wu, wd, gate, up), lambda: gated_backward(dy, x, wg, wu, wd, gate[:, :8], up),
                 lambda: gated_backward(dy.float(), x, wg, wu, wd, gate, up), lambda: gated_backward(dy, x, wg, wu, wd, gate, up.cpu()),
                 lambda: gated_forward(torch.tensor(1.0, dtype=BF, device="cuda"), wg, wu, wd)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        GatedFeedForward(8, 8, activation="tanh")


def test_in_graphs_beside_eager_calls():
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(300, 136, 264, 72)

    def call():
        y, g, u = gated_forward(x, wg, wu, wd, keep=True)
        return (y, g, u, *gated_backward(dy, x, wg, wu, wd, g, u))

    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for g in graphs:
        g.replay()
    eager = call()
    torch.cuda.synchronize()
    for out in (*outs, eager):
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("F", [72, 77, 136, 160])
@pytest.mark.parametrize("T", [5, 40, 300])
def test_kept_projections_side_by_side(T, F):
    """gate and up as halves of one matrix, through the C entry: a row ends at F, rounded up to a multiple of 8, and what is behind it stays."""
    from haste_b200 import _lib
    from haste_b200.feedforward import gated_backward, gated_forward
    x, wg, wu, wd, dy = _inputs(T, 64, F, 48)
    up8 = -(-F // 8) * 8
    kept = torch.full((T + 2, 2 * up8 + 8), 7.0, dtype=BF, device="cuda")
    gate, up, y = kept[1:-1, :up8], kept[1:-1, up8:2 * up8], torch.empty(T, 48, dtype=BF, device="cuda")
    need = _lib.lib.haste_gated_forward_scratch(T, 64, F, 48, 0)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.lib.haste_gated_forward(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), gate.data_ptr(), up.data_ptr(), y.data_ptr(), scratch.data_ptr(), need, T, 64, F, 48, 64,
                                        kept.stride(0), _lib.ACTIVATIONS["silu"], stream) == _lib.OK
    want = gated_forward(x, wg, wu, wd, keep=True)
    assert torch.equal(y, want[0]) and torch.equal(gate[:, :F], want[1]) and torch.equal(up[:, :F], want[2])
    assert (kept[0] == 7).all() and (kept[-1] == 7).all() and (kept[:, 2 * up8:] == 7).all()
    kept[:, 2 * up8:] = float("nan")                                       # and what is behind a row that is read does not count
    grads, from_halves = gated_backward(dy, x, wg, wu, wd, *want[1:]), gated_backward(dy, x, wg, wu, wd, gate[:, :F], up[:, :F])
    assert all(torch.equal(a, b) for a, b in zip(grads, from_halves))


@pytest.mark.parametrize("sizes", [(72, 136, 40), (77, 131, 33), (1, 1, 1), (64, 2104, 24), (1160, 40, 2400), (513, 65, 17)])
@pytest.mark.parametrize("T", [2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33])
def test_few_rows(T, sizes):
    """Around the steps of the forms for few rows: values, kept projections, rows that do not depend on their neighbours, whatever these hold."""
    from haste_b200.feedforward import gated_forward
    x, wg, wu, wd, _ = _inputs(T, *sizes)
    got = gated_forward(x, wg, wu, wd, "gelu_tanh", keep=True)
    _check(("y", "gate", "up"), got, *eo.gated(x, wg, wu, wd, "gelu_tanh"))
    spoilt = x.clone()
    spoilt[T // 2] = float("nan")
    spoilt[0, -1] = float("inf")
    y = gated_forward(spoilt, wg, wu, wd, "gelu_tanh")
    others = [t for t in range(T) if t not in (0, T // 2)]
    assert y[T // 2].isnan().all() and not y[0].isfinite().all() and torch.equal(y[others], got[0][others])


@pytest.mark.parametrize("T", [16, 17, 32])
def test_few_rows_of_many_weights(T):
    """Where the tiled form takes over earlier."""
    from haste_b200.feedforward import gated_forward
    x, wg, wu, wd, _ = _inputs(T, 2304, 11264, 1536)
    _check(("y", "gate", "up"), gated_forward(x, wg, wu, wd, "silu", keep=True), *eo.gated(x, wg, wu, wd, "silu"))

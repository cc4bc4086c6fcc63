"""Layer norm kernels against the 64-bit oracle, elementwise within bounds that follow from fp32 sums (oracle/dense_oracle.py), and
against differences; widths, types, strides and values at which a row kernel can go wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do

BF, F32 = torch.bfloat16, torch.float32
TYPES = [(BF, BF), (BF, F32), (F32, F32), (F32, BF)]
SHAPES = [(1, 1), (3, 1), (1, 768), (5, 7), (17, 33), (64, 768), (33, 1021), (130, 1024), (7, 4096), (9, 8200), (2, 40001), (1200, 96), (3, 31), (6, 2056),
          (11, 520), (700, 8), (5, 16384), (2, 33000)]


def _inputs(rows, D, xt, wt, seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed * 7919 + rows * 131 + D)
    x = torch.randn(rows, D, generator=gen) * torch.rand(rows, 1, generator=gen) * 3 + torch.randn(D, generator=gen)
    w, b = 1 + 0.3 * torch.randn(D, generator=gen), 0.2 * torch.randn(D, generator=gen)
    dy = torch.randn(rows, D, generator=gen) * 0.1
    return x.to(xt).to(device), w.to(wt).to(device), b.to(wt).to(device), dy.to(device)


def _check_forward(x, w, b, eps, got):
    want, tol = do.layer_norm(x, w, b, eps)
    for name, g, v, t in zip(("y", "mean", "rstd"), got, want, tol):
        assert g.shape == v.shape, name
        bad = do.outside(g, v, t, name)
        assert bad is None, bad


def _check_backward(dy, x, w, mean, rstd, got):
    want, tol = do.layer_norm_grad(dy, x, w, mean, rstd)
    for name, g, v, t in zip(("dx", "dw", "db"), got, want, tol):
        assert g.shape == v.shape, name
        bad = do.outside(g, v, t, name)
        assert bad is None, bad


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, types):
    from haste_b200.norm import layer_norm_forward
    x, w, b, _ = _inputs(*shape, *types)
    got = layer_norm_forward(x, w, b, 1e-5)
    assert got[0].dtype == x.dtype and got[1].dtype == got[2].dtype == F32
    _check_forward(x, w, b, 1e-5, got)
    assert torch.equal(layer_norm_forward(x, w, b, 1e-5, stats=False), got[0])


@pytest.mark.parametrize("dy_type", [BF, F32])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, types, dy_type):
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x, w, b, dy = _inputs(*shape, *types)
    dy = dy.to(dy_type)
    _, mean, rstd = layer_norm_forward(x, w, b, 1e-5)
    got = layer_norm_backward(dy, x, w, mean, rstd)
    assert got[0].dtype == x.dtype and got[1].dtype == got[2].dtype == w.dtype
    _check_backward(dy, x, w, mean, rstd, got)
    again = layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip(got, again))              # the order of every sum depends on the sizes alone


@pytest.mark.parametrize("rows,D", [(4096 + 3, 256), (20000, 40), (3000, 1021), (1500, 4096)])
def test_backward_of_many_rows(rows, D):
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x, w, b, dy = _inputs(rows, D, BF, F32)
    _, mean, rstd = layer_norm_forward(x, w, b, 1e-5)
    dy = dy.to(BF)
    _check_backward(dy, x, w, mean, rstd, layer_norm_backward(dy, x, w, mean, rstd))


@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("D", [768, 1021])
def test_without_weight_or_bias(D, xt):
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x, w, b, dy = _inputs(37, D, xt, F32)
    dy = dy.to(xt)
    for ww, bb in ((None, None), (w, None), (None, b)):
        got = layer_norm_forward(x, ww, bb, 1e-3)
        _check_forward(x, ww, bb, 1e-3, got)
        grads = layer_norm_backward(dy, x, ww, got[1], got[2])
        assert grads[1].dtype == (xt if ww is None else F32)
        _check_backward(dy, x, ww, got[1], got[2], grads)
    dx, dw, db = layer_norm_backward(dy, x, w, got[1], got[2], want_weight=False, want_bias=False)
    assert dw is None and db is None and torch.equal(dx, layer_norm_backward(dy, x, w, got[1], got[2])[0])
    dx, dw, db = layer_norm_backward(dy, x, w, got[1], got[2], want_weight=False)
    assert dw is None and torch.equal(db, layer_norm_backward(dy, x, w, got[1], got[2])[2])


@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("D", [1, 24, 768, 1021])
def test_strides_and_alignment(D, xt):
    """Rows inside wider ones, at every offset from a 16-byte boundary; transposed, repeated, cut and reversed leading dimensions."""
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    gen = torch.Generator(device="cuda").manual_seed(D)
    wide = torch.randn(13, D + 40, generator=gen, device="cuda").to(xt)
    wbuf = torch.randn(2, D + 8, generator=gen, device="cuda")
    cases = [wide[:, o:o + D] for o in (0, 1, 2, 3, 5, 8)] + [wide[::2, 4:4 + D], wide[:D, :13].t() if D <= 13 else wide[:1, 7:7 + D].expand(9, D)]
    cases += [torch.randn(D, 6, generator=gen, device="cuda").to(xt).t(), torch.randn(4, 3, D, generator=gen, device="cuda").to(xt).transpose(0, 1),
              torch.randn(4, 3, D + 1, generator=gen, device="cuda").to(xt)[:, 1:, :D], torch.randn(D, generator=gen, device="cuda").to(xt)]
    for k, x in enumerate(cases):
        w, b = wbuf[0, k % 4:k % 4 + D], wbuf[1, (k + 1) % 5:(k + 1) % 5 + D]
        got = layer_norm_forward(x, w, b, 1e-5)
        _check_forward(x, w, b, 1e-5, got)
        for dy in (torch.randn(x.shape, generator=gen, device="cuda").to(xt), torch.randn(D, generator=gen, device="cuda").expand(x.shape),
                   torch.randn(1, generator=gen, device="cuda").to(BF).expand(x.shape)):
            _check_backward(dy, x, w, got[1], got[2], layer_norm_backward(dy, x, w, got[1], got[2]))


@pytest.mark.parametrize("D", [768, 1021, 9000])
def test_no_rows(D):
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x = torch.empty(0, 3, D, device="cuda", dtype=BF)
    w = torch.ones(D, device="cuda")
    y, mean, rstd = layer_norm_forward(x, w, w)
    assert y.shape == x.shape and mean.shape == rstd.shape == (0, 3)
    dx, dw, db = layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == x.shape and not dw.any() and not db.any() and dw.shape == db.shape == (D,)


@pytest.mark.parametrize("D", [8, 768, 1021, 4096, 9000])
def test_rows_of_unusual_values(D):
    """Constant rows (variance 0), rows far from zero against their spread, very small and very large ones; an inf or NaN stays in its row."""
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x, w, b, dy = _inputs(12, D, F32, F32)
    x[0] = 0.0
    x[1] = 123.0
    x[2] = 4096.0 + x[2] * 0.01
    x[3] *= 1e-20
    x[4] *= 1e15
    x[5] = 1e-30
    got = layer_norm_forward(x, w, b, 1e-5)
    _check_forward(x, w, b, 1e-5, got)
    assert torch.equal(got[0][0], b) and torch.equal(got[0][1], b)
    _check_backward(dy, x, w, got[1], got[2], layer_norm_backward(dy, x, w, got[1], got[2]))
    grads = layer_norm_backward(dy, x, w, got[1], got[2])
    spoilt = x.clone()
    spoilt[7, D // 2] = float("nan")
    spoilt[9, 0] = float("inf")
    spoilt[10, D - 1] = float("-inf")
    y, mean, rstd = layer_norm_forward(spoilt, w, b, 1e-5)
    keep = torch.tensor([i not in (7, 9, 10) for i in range(12)], device="cuda")
    assert torch.equal(y[keep], got[0][keep]) and bool(y[~keep].isnan().any(1).all())
    dx, _, db = layer_norm_backward(dy, spoilt, w, mean, rstd)
    assert torch.equal(dx[keep], grads[0][keep]) and bool(dx[~keep].isnan().any(1).all()) and torch.equal(db, grads[2])


@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("value", [torch.finfo(BF).min, torch.finfo(BF).max])
@pytest.mark.parametrize("D", [1, 2, 4, 16, 64, 1024, 2048, 16384])
def test_rows_of_the_largest_numbers(D, value, xt):
    """A constant row has itself as mean, variance 0, z = 0: y = b and dx = r (h - mean(h)), however large the constant is.  Where D is a power of two
    and the constant has 8 significant bits, every partial sum is exact."""
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x, w, b, dy = _inputs(9, D, xt, F32)
    x[1::2] = value
    dy = dy.to(F32)
    y, mean, rstd = layer_norm_forward(x, w, b, 1e-5)
    big = slice(1, None, 2)
    assert torch.equal(y[big], b.to(xt).expand_as(y[big])) and bool((mean[big] == value).all())
    assert bool(((rstd[big].double() - 1e-5 ** -0.5).abs() <= 6 * do.U * 1e-5 ** -0.5).all())      # eps, its root and the quotient rounded
    dx, dw, db = layer_norm_backward(dy, x, w, mean, rstd)
    h, r = dy[big].double() * w.double(), rstd[big].double()[:, None]
    mh = h.mean(-1, keepdim=True)
    tol = r * (4 * do.U * (h.abs() + mh.abs()) + do.chain(D) * h.abs().mean(-1, keepdim=True))
    bad = do.outside(dx[big], r * (h - mh), tol, "dx")
    assert bad is None, bad
    # the other rows have what they would have alone, and the large ones add nothing to dw
    alone = layer_norm_backward(dy[::2].contiguous(), x[::2].contiguous(), w, mean[::2].contiguous(), rstd[::2].contiguous())
    assert torch.equal(dx[::2], alone[0]) and bool(torch.isfinite(dw).all())
    want, tol = do.layer_norm_grad(dy[::2], x[::2], w, mean[::2], rstd[::2])
    bad = do.outside(dw, want[1], tol[1], "dw") or do.outside(db, dy.double().sum(0), 73 * do.U * dy.double().abs().sum(0), "db")
    assert bad is None, bad


@pytest.mark.parametrize("D", [40, 768, 1021])
def test_gradients_against_differences(D):
    """Directional derivatives of sum(y * dy) by central differences of the forward kernel.  With steps of 2^-7 in directions of unit size
    the third-order term is below 2^-14 of the derivatives' scale, the fp32 rounding of y below 2^-24 / 2^-7 times sqrt(n)."""
    from haste_b200.norm import layer_norm
    x, w, b, dy = _inputs(6, D, F32, F32)
    x = x / x.std(1, keepdim=True)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    layer_norm(*leaves, 1e-5).backward(dy)
    gen = torch.Generator(device="cuda").manual_seed(5)
    f = lambda *t: float((layer_norm(*t, 1e-5).double() * dy.double()).sum())
    h = 2.0 ** -7
    for k in range(3):
        d = torch.randn(leaves[k].shape, generator=gen, device="cuda")
        args = lambda s: [t.detach() + (s * h * d if i == k else 0) for i, t in enumerate(leaves)]
        with torch.no_grad():
            slope = (f(*args(1)) - f(*args(-1))) / (2 * h)
        scale = float(leaves[k].grad.double().norm())                     # of a derivative in a random direction
        assert abs(slope - float((leaves[k].grad.double() * d.double()).sum())) <= 2e-3 * scale, k


def test_module_and_autograd():
    from haste_b200.norm import LayerNorm
    ref = torch.nn.LayerNorm(768, device="cuda")
    with torch.no_grad():
        ref.weight.normal_(1, 0.2)
        ref.bias.normal_(0, 0.2)
    m = LayerNorm(768, device="cuda")
    m.load_state_dict(ref.state_dict())
    x = torch.randn(4, 9, 768, device="cuda", dtype=BF)
    with torch.no_grad():
        y0 = m(x)
    xg = x.clone().requires_grad_(True)
    y = m(xg)
    assert torch.equal(y, y0) and y.dtype == BF
    _check_forward(x, m.weight.detach(), m.bias.detach(), 1e-5, (y.detach(),) + tuple(s.float() for s in do.layer_norm(x, None, None, 1e-5)[0][1:]))
    y.sum().backward()                                                     # a broadcast gradient
    _, mean, rstd = do.layer_norm(x, None, None, 1e-5)[0]
    want, tol = do.layer_norm_grad(torch.ones_like(x), x, m.weight.detach(), mean, rstd)
    tol_s = do.layer_norm(x, None, None, 1e-5)[1]
    # the statistics are the kernel's, in fp32: a relative error of rstd and an error of the mean enter dx and dw to first order
    rel = (tol_s[2] / rstd)[..., None] + do.U
    z = (x.double() - mean[..., None]) * rstd[..., None]
    ez = (tol_s[1] * rstd)[..., None] + z.abs() * rel + do.U * z.abs()
    h = m.weight.detach().double()
    dx_tol = tol[0] + rstd[..., None] * (ez * (h * z).mean(-1, keepdim=True).abs() + z.abs() * (h.abs() * ez).mean(-1, keepdim=True)) + 3 * rel * want[0].abs()
    assert do.outside(xg.grad, want[0], dx_tol, "dx") is None
    assert do.outside(m.weight.grad, want[1], tol[1] + ez.reshape(-1, 768).sum(0), "dw") is None
    assert do.outside(m.bias.grad, want[2], tol[2], "db") is None
    assert LayerNorm(8, bias=False, device="cuda").bias is None
    # only what is asked for
    w = m.weight.detach()
    only = x.clone().requires_grad_(True)
    from haste_b200.norm import layer_norm
    layer_norm(only, w, None).backward(torch.ones_like(x))
    assert only.grad is not None and w.grad is None
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(layer_norm(only, w, None).float().square().sum(), only, create_graph=True)[0]
        g.sum().backward()


def test_on_another_stream_and_in_a_graph():
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    x, w, b, dy = _inputs(300, 768, BF, F32)
    dy = dy.to(BF)
    want = layer_norm_forward(x, w, b)
    grads = layer_norm_backward(dy, x, w, *want[1:])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layer_norm_forward(x, w, b)
        grads2 = layer_norm_backward(dy, x, w, *got[1:])
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want + grads, got + grads2))
    g = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(g):
        out = layer_norm_forward(xs, w, b)
        grads3 = layer_norm_backward(dy, xs, w, *out[1:])
    for seed in (1, 2):
        x2 = _inputs(300, 768, BF, F32, seed)[0]
        xs.copy_(x2)
        g.replay()
        torch.cuda.synchronize()
        again = layer_norm_forward(x2, w, b)
        assert all(torch.equal(a, c) for a, c in zip(out + grads3, again + layer_norm_backward(dy, x2, w, *again[1:])))


def test_more_than_2_31_elements():
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    D = 1024
    rows = 2 ** 31 // D + 5
    x = torch.empty(rows, D, device="cuda", dtype=BF)
    x[:8].normal_()
    x[8:-8] = 1.0
    x[-8:].normal_()
    w, b = torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda")
    y, mean, rstd = layer_norm_forward(x, w, b)
    for part in (slice(0, 8), slice(rows - 8, rows)):
        _check_forward(x[part], w, b, 1e-5, (y[part], mean[part], rstd[part]))
    del y
    dy = torch.zeros(rows, D, device="cuda", dtype=BF)
    dy[:8].normal_()
    dy[-8:].normal_()
    dx, dw, db = layer_norm_backward(dy, x, w, mean, rstd)
    ends = torch.cat([torch.arange(8), torch.arange(rows - 8, rows)]).cuda()
    _check_backward(dy[ends], x[ends], w, mean[ends], rstd[ends], (dx[ends], dw, db))


def test_refusals():
    from haste_b200 import _lib
    from haste_b200.norm import layer_norm, layer_norm_backward, layer_norm_forward
    x, w = torch.randn(4, 16, device="cuda"), torch.ones(16, device="cuda")
    y, mean, rstd = layer_norm_forward(x, w, w)
    bad = [lambda: layer_norm(x.half(), w, w), lambda: layer_norm(x, w.half(), None), lambda: layer_norm(x, w, w.to(BF)), lambda: layer_norm(x, w[:8], None),
           lambda: layer_norm(x, w.cpu(), None), lambda: layer_norm(x.cpu(), w, w), lambda: layer_norm(x[:, :0], None, None), lambda: layer_norm(x, w, None, -1.0),
           lambda: layer_norm(x, w, None, float("nan")), lambda: layer_norm(x, torch.ones(32, device="cuda")[::2], None), lambda: layer_norm(x, w[None], None),
           lambda: layer_norm_backward(y[:2], x, w, mean, rstd), lambda: layer_norm_backward(y, x, w, mean[:2], rstd), lambda: layer_norm_backward(y, x, w, mean.to(BF), rstd),
           lambda: layer_norm_backward(y.half(), x, w, mean, rstd), lambda: layer_norm_backward(y, x, w, mean, rstd, param_dtype=BF),
           lambda: layer_norm_backward(y.cpu(), x, w, mean, rstd)]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was not refused")
    assert _lib.lib.haste_poll_status() == _lib.OK


@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("D", [2, 12, 16, 72, 96, 101, 192, 257, 333, 384, 500, 513, 767, 1017, 1018, 1023, 1025, 2047, 4093, 8191, 16383])
def test_groups_of_lanes_and_vectors(D, xt):
    """Widths between which a row changes its lanes, vectors or block, with more rows than one turn of the groups takes where that is cheap."""
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    rows = 9001 if D <= 192 else 2311 if D <= 1025 else 83
    x, w, b, dy = _inputs(rows, D, xt, BF)
    dy = dy.to(xt)
    got = layer_norm_forward(x, w, b, 1e-5)
    _check_forward(x, w, b, 1e-5, got)
    _check_backward(dy, x, w, got[1], got[2], layer_norm_backward(dy, x, w, got[1], got[2]))

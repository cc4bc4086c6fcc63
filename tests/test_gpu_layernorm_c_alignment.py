"""The C entry points with outputs that lie one element off a 16-byte boundary: nothing needs alignment beyond that of its type, and nothing
is written outside the outputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do

BF, F32 = torch.bfloat16, torch.float32
GUARD = 64


def _guarded(rows, D, dtype):
    """A buffer of a value that no result has, and the output inside it, one element off."""
    buf = torch.full((rows * D + 2 * GUARD + 1,), 12345.0, device="cuda", dtype=dtype)
    return buf, buf[GUARD + 1:GUARD + 1 + rows * D].view(rows, D)


def _untouched(buf, n):
    keep = torch.full((1,), 12345.0, device="cuda", dtype=buf.dtype)
    return bool((buf[:GUARD + 1] == keep).all()) and bool((buf[GUARD + 1 + n:] == keep).all())


@pytest.mark.parametrize("wt", [BF, F32])
@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("rows,D", [(1, 1), (7, 24), (130, 768), (33, 1021), (1100, 100)])
def test_outputs_off_the_boundary(rows, D, xt, wt):
    from haste_b200 import _lib
    gen = torch.Generator(device="cuda").manual_seed(rows * D)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, w, b, dy = rnd(rows, D).to(xt), (1 + 0.3 * rnd(D)).to(wt), rnd(D).to(wt), rnd(rows, D).to(xt)
    kind = {BF: _lib.BF16, F32: _lib.FP32}
    st = torch.cuda.current_stream().cuda_stream
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    buf, y = _guarded(rows, D, xt)
    _lib.check(_lib.lib.haste_layer_norm_forward(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), rows, D, D, 1e-5,
                                                 kind[xt], kind[wt], st), "forward")
    want, tol = do.layer_norm(x, w, b, 1e-5)
    for name, got, v, t in zip(("y", "mean", "rstd"), (y, mean, rstd), want, tol):
        bad = do.outside(got, v, t, name)
        assert bad is None, bad
    assert _untouched(buf, rows * D)
    buf, dx = _guarded(rows, D, xt)
    size = _lib.lib.haste_layer_norm_backward_scratch(rows, D)
    scratch = torch.full((size + 256,), 77, device="cuda", dtype=torch.uint8)
    params = [_guarded(1, D, wt) for _ in range(2)]
    _lib.check(_lib.lib.haste_layer_norm_backward(dy.data_ptr(), x.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), params[0][1].data_ptr(),
                                                  params[1][1].data_ptr(), scratch.data_ptr(), size, rows, D, D, D, kind[xt], kind[xt], kind[wt], st), "backward")
    want, tol = do.layer_norm_grad(dy, x, w, mean, rstd)
    for name, got, v, t in zip(("dx", "dw", "db"), (dx, params[0][1][0], params[1][1][0]), want, tol):
        bad = do.outside(got, v, t, name)
        assert bad is None, bad
    assert _untouched(buf, rows * D) and all(_untouched(p, D) for p, _ in params) and bool((scratch[size:] == 77).all())

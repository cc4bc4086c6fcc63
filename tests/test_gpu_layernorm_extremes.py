"""Layer norm of rows of the largest numbers of their type, whatever their number of elements and the roundings on the way."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("D", [1, 2, 3, 5, 6, 7, 12, 31, 100, 768, 1000, 1021, 1024, 2048, 4096, 8191, 9000, 20000])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("xt", [BF, F32])
def test_constant_rows_of_the_largest_number(xt, sign, D):
    """The mean of such a row is the number itself.  The computed one may be off by the roundings of its sum, but not beyond the type's range; the
    variance is then 0 or, an ulp of the number squared, inf, and y is the bias either way.  The gradients are those for the returned statistics."""
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    gen = torch.Generator().manual_seed(D)
    x = torch.randn(8, D, generator=gen)
    value = sign * torch.finfo(xt).max
    x[::2] = value
    x, w, b, dy = (t.cuda() for t in (x.to(xt), torch.rand(D, generator=gen) + 0.5, torch.randn(D, generator=gen), torch.randn(8, D, generator=gen) * 0.1))
    y, mean, rstd = layer_norm_forward(x, w, b, 1e-5)
    assert torch.equal(y[::2], b.to(xt).expand_as(y[::2]))
    assert bool(((mean[::2].double() / value - 1).abs() <= do.chain(D)).all()) and bool(torch.isfinite(rstd).all())
    (want, want_mean, want_rstd), tol = do.layer_norm(x[1::2], w, b, 1e-5)
    for got, v, t in zip((y[1::2], mean[1::2], rstd[1::2]), (want, want_mean, want_rstd), tol):
        bad = do.outside(got, v, t)
        assert bad is None, bad
    dx, dw, db = layer_norm_backward(dy, x, w, mean, rstd)
    want, tol = do.layer_norm_grad(dy, x, w, mean, rstd)
    # x - mean is 0 in the large rows, or their rstd is: they add nothing to dw
    (_, want_w, _), (_, tol_w, _) = do.layer_norm_grad(dy[1::2], x[1::2], w, mean[1::2], rstd[1::2])
    for name, got, v, t in (("dx", dx, want[0], tol[0]), ("dw", dw, want_w, tol_w), ("db", db, want[2], tol[2])):
        bad = do.outside(got, v, t, name)
        assert bad is None, bad


@pytest.mark.parametrize("D", [5, 768, 1021, 9000])
def test_a_row_with_an_infinity_stays_nan(D):
    from haste_b200.norm import layer_norm_forward
    x = torch.full((4, D), torch.finfo(F32).max, device="cuda")
    x[1, D // 2], x[2, 0], x[3, D - 1] = float("inf"), float("-inf"), float("nan")
    y, mean, rstd = layer_norm_forward(x, None, None, 1e-5)
    assert not bool(y[0].any()) and bool(y[1:].isnan().all())

"""64-bit restatements of the dense operators next to the sparse layer (test infrastructure): layer norm and its gradient.

Each returns, beside the values, what the kernels' tests derive their tolerances from.  All tensors are torch tensors on any device.
"""
import torch

U = 2.0 ** -24            # unit roundoff of fp32
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # relative error of one rounding to the type
TINIEST = {torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}    # and its absolute error among the subnormals


def chain(n):
    """Relative error bound of an fp32 sum of n terms whose partial sums are chains of at most n / 32 + 64 additions (a warp's lanes
    add their elements, then the lanes and warps are added)."""
    return (n / 32 + 64) * U


def layer_norm(x, w, b, eps):
    """(y, mean, rstd) in float64, and elementwise bounds (tol_y, tol_mean, tol_rstd) for fp32 arithmetic before y's rounding.

    mean: chain(D) times the mean of |x|.  The centred values are off by that and an ulp of themselves, the variance by twice the
    first-order part (which cancels up to chain(D), as the deviations sum to zero) plus chain(D): relative 2 chain(D) plus the square
    of the mean's error; rstd half of that plus the rounding of root and quotient."""
    x = x.double()
    D = x.shape[-1]
    mean = x.mean(-1)
    var = (x - mean[..., None]).square().mean(-1)
    rstd = (var + eps).rsqrt()
    z = (x - mean[..., None]) * rstd[..., None]
    ww = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    bb = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = z * ww + bb
    tol_mean = chain(D) * x.abs().mean(-1) + 1e-45
    rel_var = 2 * chain(D) + 4 * U + ((tol_mean + U * x.abs().amax(-1)) * rstd).square() * 4 + 4 * U * (x.abs().amax(-1) * rstd)
    tol_rstd = rstd * (rel_var + 4 * U)
    tol_z = (tol_mean[..., None] + 2 * U * x.abs()) * rstd[..., None] + z.abs() * (rel_var[..., None] + 6 * U)
    return (y, mean, rstd), (tol_z * ww.abs() + 3 * U * (y.abs() + bb.abs()), tol_mean, tol_rstd)


def layer_norm_grad(dy, x, w, mean, rstd):
    """(dx, dw, db) in float64 for the given statistics, and bounds for fp32 arithmetic before the results' rounding."""
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[..., None], rstd.double()[..., None]
    D = x.shape[-1]
    ww = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    z = (x - mean) * rstd
    ez = 2 * U * ((x.abs() + mean.abs()) * rstd + z.abs())              # z in fp32
    h = dy * ww
    mh, mhz = h.mean(-1, keepdim=True), (h * z).mean(-1, keepdim=True)
    dx = rstd * (h - mh - z * mhz)
    emh = chain(D) * h.abs().mean(-1, keepdim=True)
    emhz = (h.abs() * ez).mean(-1, keepdim=True) + chain(D) * (h * z).abs().mean(-1, keepdim=True)
    tol_dx = rstd * (4 * U * (h.abs() + mh.abs() + (z * mhz).abs()) + emh + z.abs() * emhz + ez * mhz.abs())
    flat = lambda t: t.reshape(-1, D)
    rows = flat(x).shape[0]
    dw, db = flat(dy * z).sum(0), flat(dy).sum(0)
    # rows are added one after the other by a thread at worst
    tol_w = flat(dy.abs() * ez).sum(0) + (rows + 64) * U * flat((dy * z).abs()).sum(0)
    tol_b = (rows + 64) * U * flat(dy.abs()).sum(0)
    return (dx, dw, db), (tol_dx, tol_w, tol_b)


def outside(got, want, tol, what=""):
    """The worst value of ``got`` against ``want`` +- (``tol`` and one rounding to got's type), as a message; None if all are inside."""
    g = got.double()
    allow = tol + HALF_ULP[got.dtype] * (want.abs() + tol) + TINIEST[got.dtype]
    off = (g - want).abs()
    bad = ~(off <= allow)
    if not bool(bad.any()):
        return None
    i = int(torch.where(bad, off / allow, torch.zeros_like(off)).nan_to_num(1e300).argmax()) if off.numel() else 0
    return f"{what}: {int(bad.sum())} of {off.numel()} outside, worst at {i}: {g.reshape(-1)[i]:.9g} for {want.reshape(-1)[i]:.9g} +- {allow.expand_as(off).reshape(-1)[i]:.3g}"

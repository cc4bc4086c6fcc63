"""64-bit restatements of the dense operators next to the sparse layer (test infrastructure): layer norm and its gradient, AdamW with
moments in 32 or 8 bits.

Each returns, beside the values, what the kernels' tests derive their tolerances from.  All tensors are torch tensors on any device.
"""
import math

import numpy as np
import torch

from .philox import philox4x32

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


# ------------------------------------------------------------------ AdamW
BLOCK, TOP = 256, 1.875
M_CODES = [0.0] + [math.ldexp(1 + (c % 8) / 8, c // 8 - 15) for c in range(1, 128)]
M_CODES += [-v for v in M_CODES]
V_CODES = [0.0] + [math.ldexp(1 + (c % 8) / 8, c // 8 - 31) for c in range(1, 256)]


def random_words(n, seed, step, stream=0, first=0):
    """The 32 random bits of elements first .. first+n-1 of the moments (first a multiple of 4): uint32 [n]."""
    i = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    return np.stack(philox4x32(i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), stream, 1, seed, step, rounds=7), 1).reshape(-1)[:n]


def decode(codes, scales, signed):
    table = torch.tensor(M_CODES if signed else V_CODES, dtype=torch.float64)
    return table[codes.long()] * scales.double().repeat_interleave(BLOCK)


def code_position(y, signed):
    """Where |y| (float64, at most 1.875) lies on the scale of codes: code c at c, linear between codes; -inf for 0."""
    m, e = torch.frexp(y.abs())                                         # |y| = m 2^e, m in [0.5, 1)
    pos = 8.0 * (e.double() - 1 + (15 if signed else 31)) + 8.0 * (2 * m - 1)
    return torch.where(y == 0, torch.full_like(pos, -math.inf), pos)


def check_codes(codes, scales, x, tol, r8, signed, what=""):
    """Codes and scales of float64 values x that the kernel had to within tol: the scale is the block's largest value / 1.875, and each
    code is floor(position + (r8 + 1/2) / 256), or its neighbour where the position is too near to a whole number to tell.  None if so."""
    top, ttop = x.view(-1, BLOCK).abs().amax(1), tol.view(-1, BLOCK).amax(1)
    zero = top < 2.0 ** -121
    off = (scales.double() - torch.where(zero, 0.0, top / TOP)).abs()
    sure = zero | (top > 2.0 ** -119)
    if bool((off > ttop + 4 * U * top)[sure].any()):
        return f"{what}: a scale is off by {float(off.max())}"
    s = scales.double().repeat_interleave(BLOCK)
    live = s > 0
    y = torch.where(live, x / torch.where(live, s, 1.0), 0.0)
    rel = torch.where(live, tol / torch.where(live, s, 1.0), 0.0) + 8 * U * y.abs()
    shift = (r8.double() + 0.5) / 256
    most = 127 if signed else 255
    lo, hi = ((code_position((y.abs() + d).clamp(min=0.0), signed) + shift).floor().clamp(0 if signed else 1, most) for d in (-rel, rel))
    got = codes.long()
    mag = got % 128 if signed else got
    lo = torch.where(y.abs() <= rel, 0.0, lo)                           # may have been zero
    hi = torch.where((y == 0) & (rel == 0), 0.0, hi)
    bad = (mag < lo) | (mag > hi) | (~live & (got != 0))
    if signed:
        bad |= (mag > 0) & ((got > 127) != (x < 0)) & (y.abs() > rel)
    if bool(bad.any()):
        i = int(bad.nonzero()[0])
        return f"{what}: {int(bad.sum())} of {bad.numel()} codes, first {i}: {int(got[i])} for {float(y[i]):.9g}, {float(lo[i])} .. {float(hi[i])}"
    return None


def adamw(w, g, m, v, step, lr, b1, b2, eps, wd, scale=1.0):
    """((w', m', v'), tolerances of fp32 arithmetic) in float64."""
    w, g, m, v = (t.double() for t in (w, g, m, v))
    g = g * scale
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    tol_m = 8 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + 1e-44
    tol_v = 12 * U * v1 + 1e-44
    rate = lr / (1 - b1 ** step)
    den = v1.sqrt() / math.sqrt(1 - b2 ** step) + eps
    w1 = w * (1 - lr * wd) - rate * m1 / den
    # v below the fp32 subnormals' step leaves the root off by the root of that
    rel_den = 16 * U + (tol_v.sqrt() / math.sqrt(1 - b2 ** step) / den).clamp(max=1.0) * (v1 < 1e-37)
    return (w1, m1, v1), (4 * U * (w.abs() + w1.abs()) + rate / den * (tol_m + m1.abs() * rel_den), tol_m, tol_v)


def stochastic_bf16(w, r16):
    """float64 values rounded to bf16 with 16 random bits: the fp32 pattern plus the bits, cut."""
    bits = w.float().view(torch.int32).to(torch.int64) & 0xFFFFFFFF
    bits = (bits + r16.to(torch.int64)) & 0xFFFF0000
    bits = torch.where(bits > 0x7FFFFFFF, bits - (1 << 32), bits)
    return bits.to(torch.int32).view(torch.float32)


def check_bf16(got, w, tol, r16, what=""):
    """Stochastically rounded weights: between those of w - tol and w + tol (rounding is monotone in the size of w).  r16 None: to nearest."""
    a = tol + U * w.abs() + 1e-44
    if r16 is None:
        ends = [(w + d).bfloat16().float() for d in (-a, a)]
    else:
        ends = [stochastic_bf16(w + d, r16) for d in (-a, a)]
        cross = (w - a <= 0) & (w + a >= 0)                             # the sign is open: anything near zero
        ends = [torch.where(cross, -1.01 * a.float() - 1e-40, ends[0]), torch.where(cross, 1.01 * a.float() + 1e-40, ends[1])]
    bad = ~((got.float() >= ends[0]) & (got.float() <= ends[1]))
    if bool(bad.any()):
        i = int(bad.nonzero()[0])
        return f"{what}: {int(bad.sum())} of {bad.numel()} weights, first {i}: {float(got[i])} for {float(w[i]):.9g} +- {float(a[i]):.3g}"
    return None

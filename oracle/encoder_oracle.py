"""64-bit restatements of the operators of an encoder in front of the sparse layer (test infrastructure): token embedding and its gradient, the gated
feed-forward block and its gradients, Newton-Schulz steps and the Muon update.

Each returns, beside the values, what the kernels' tests derive their tolerances from.  All tensors are torch tensors on any device.
"""
import math

import torch

from .dense_oracle import U, outside  # noqa: F401

A, B, C = 3.4445, -4.7750, 2.0315


# ------------------------------------------------------------------ token embedding
def embedding(ids, table, scale):
    """(y, bound before its rounding): one fp32 product."""
    ok = (ids >= 0) & (ids < table.shape[0])
    y = table.double()[ids.clamp(0, table.shape[0] - 1).long()] * float(torch.tensor(scale, dtype=torch.float32))
    return torch.where(ok[..., None], y, torch.full_like(y, math.nan)), U * y.abs()


def embedding_grad(dy, ids, rows, scale, padding=None):
    """(dtable, bound): a row of n tokens is a chain of at most n additions in whatever parts, each off by U of its partial sum, and a product."""
    D = dy.shape[-1]
    ids, dy = ids.reshape(-1).long(), dy.reshape(-1, D).double()
    keep = (ids >= 0) & (ids < rows) & (ids != (-1 if padding is None else padding % rows))
    s = float(torch.tensor(scale, dtype=torch.float32))
    zeros = torch.zeros(rows, D, dtype=torch.float64, device=dy.device)
    total, size = zeros.index_add(0, ids[keep], dy[keep]), zeros.index_add(0, ids[keep], dy[keep].abs())
    n = torch.bincount(ids[keep], minlength=rows).double()
    return total * s, ((n + 2) * U)[:, None] * size * abs(s)


# ------------------------------------------------------------------ gated feed-forward block
def activation(g, kind):
    """(act, act', relative bound of fp32 arithmetic for either, in units of U): what exp, erfc or a cubic add to a few roundings is proportional to their argument's size."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 24 + 8 * g.abs()
    if kind == "relu":
        return g.clamp(min=0), (g > 0).double(), torch.zeros_like(g)
    if kind == "gelu":
        cdf = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        pdf = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        return g * cdf, cdf + g * pdf, 24 + 8 * g * g
    k = 2 * math.sqrt(2 / math.pi)
    arg = k * (g + 0.044715 * g ** 3)
    s = torch.sigmoid(arg)
    return g * s, s + g * s * (1 - s) * k * (1 + 3 * 0.044715 * g * g), 24 + 16 * arg.abs()


def _rounded(v, tol):
    """v in bf16 (as fp64), and how far a value within tol of it may be from that once rounded: 0 unless a border between two bf16 lies there."""
    r = lambda x: x.float().to(torch.bfloat16).double()
    mid = r(v)
    return mid, torch.maximum((r(v + tol) - mid).abs(), (r(v - tol) - mid).abs())


def _product(a, ea, b, spec):
    """(sum of a b, bound) with errors ea of a; n fp32 additions, each off by 2 U of the partial sum's size at most (tensor cores truncate)."""
    value, size = torch.einsum(spec, a, b), torch.einsum(spec, a.abs(), b.abs())
    inner = set(spec.split("->")[0].replace(",", "")) - set(spec.split("->")[1])
    n = 1
    for c in inner:
        left = spec.split(",")[0]
        n *= a.shape[left.index(c)]
    bound = 2 * (n + 32) * U * size
    if ea is not None:
        bound = bound + torch.einsum(spec, ea, b.abs())
    return value, bound


def gated(x, wg, wu, wd, kind, few=8):
    """((y, gate, up), bounds): h is rounded to bf16 unless there are `few` rows at most."""
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    gate, eg = _product(x, None, wg, "td,fd->tf")
    up, eu = _product(x, None, wu, "td,fd->tf")
    a, slope, units = activation(gate, kind)
    # act is Lipschitz: |act'| < 1.13 for all of them
    ea = 1.13 * eg + units * U * a.abs() + 1e-35
    h = a * up
    eh = ea * (up.abs() + eu) + a.abs() * eu + 2 * U * h.abs()
    if x.shape[0] > few:
        h, eh = _rounded(h, eh)
    y, ey = _product(h, eh, wd, "tf,of->to")
    return (y, gate, up), (ey, eg, eu)


def gated_grad(dy, x, wg, wu, wd, gate, up, kind):
    """((dx, dwg, dwu, dwd), bounds) from the kept projections; dgate, dup and h are rounded to bf16."""
    dy, x, wg, wu, wd, gate, up = (t.double() for t in (dy, x, wg, wu, wd, gate, up))
    dh, ed = _product(dy, None, wd, "to,of->tf")
    a, slope, units = activation(gate, kind)
    ea, es = units * U * a.abs() + 1e-35, units * U * (slope.abs() + a.abs() + 1e-3) + 1e-35
    dgate, dup = dh * up * slope, dh * a
    dgate, e1 = _rounded(dgate, ed * (up * slope).abs() + (dh * up).abs() * es + ed * up.abs() * es + 4 * U * dgate.abs())
    dup, e2 = _rounded(dup, ed * a.abs() + (dh.abs() + ed) * ea + 4 * U * dup.abs())
    h, e3 = _rounded(a * up, ea * up.abs() + 2 * U * (a * up).abs())
    one, b1 = _product(dgate, e1, wg, "tf,fd->td")
    two, b2 = _product(dup, e2, wu, "tf,fd->td")
    dwg, b3 = _product(dgate, e1, x, "tf,td->fd")
    dwu, b4 = _product(dup, e2, x, "tf,td->fd")
    dwd, b5 = _product(h, e3, dy, "tf,to->of")
    # (the two sums of dx are one chain)
    return (one + two, dwg, dwu, dwd), (2 * (b1 + b2), b3, b4, b5)


# ------------------------------------------------------------------ Newton-Schulz steps
def orthogonalize(g, steps=5, coefficients=(A, B, C), eps=1e-7):
    """The definition in 64 bits."""
    a, b, c = coefficients
    tall = g.shape[0] > g.shape[1]
    x = g.double()
    x = (x.t() if tall else x) / max(float(x.norm()), eps)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


def orthogonalize_rounded(g, steps=5, coefficients=(A, B, C), eps=1e-7):
    """The same with the kernels' roundings and no others: products take X (times 256), A and B = a I + b A + c A^2 in fp16; X has 11 more bits, which a
    alone multiplies, in the first step and up to the last but two."""
    a, b, c = coefficients
    f16 = lambda v: v.to(torch.float16).double()
    tall = g.shape[0] > g.shape[1]
    x = g.double()
    x = (x.t() if tall else x) / max(float(x.norm()), eps) * 256
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for k in range(steps):
        hi = f16(x)
        low = f16((x - hi) * 2048) / 2048 if k == 0 or k < steps - 2 else torch.zeros_like(x)
        s = f16(hi @ hi.t() / 65536)
        x = f16(a * eye + b * s + c * (s @ s)) @ hi + a * low
    x = f16(x) / 256
    return x.t() if tall else x


def orthogonalize_bound(g, steps=5, coefficients=(A, B, C), eps=1e-7):
    """(exact result, bound of the 2-norm of a kernel's error): three times what the roundings above make of it (the kernel's sums are fp32, so near a border it rounds to the other
    side, which is another error of the same size), and the result's own rounding to bf16, 2^-8 of each value at most."""
    exact = orthogonalize(g, steps, coefficients, eps)
    off = float((orthogonalize_rounded(g, steps, coefficients, eps) - exact).norm())
    return exact, 3 * off + 2.0 ** -8 * float(exact.norm()) + 1e-30


def muon_rate(shape, lr, adjust):
    return lr * (0.2 * math.sqrt(max(shape)) if adjust == "match_rms_adamw" else math.sqrt(max(1.0, shape[0] / shape[1])))

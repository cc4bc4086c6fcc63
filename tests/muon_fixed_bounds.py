"""What Newton-Schulz steps may be off by against their 64-bit definition, whatever the kernel rounds on its way.

Rounding to nearest is off by u = eps / 2 of a value at most, and by 0.43 u in the root mean square over values spread evenly between two powers of two: 1.7e-3 for the result in bf16 (u = 2^-8), 2.1e-4
where something is rounded to fp16 (u = 2^-11).  A step maps a singular value s to s (a + b s^2 + c s^4).  For s up to 1 it multiplies an error of X by |a + 3 b s^2 + 5 c s^4|, 3.4445 at most, one of
A by |b + 2 c s^2| s, 2.0 at most, and one of B counts as one of what the step makes.  With fp16 products that gives in the end, as parts of the result, at most: X before the last step but one
2.1e-4 3.4445^2 = 2.5e-3, before the last 0.7e-3; A 1.4e-3 and 0.4e-3, B 0.7e-3 and 0.2e-3; the result's own rounding 1.7e-3; in squares 3.5e-3.  (What is rounded in steps before these lies mostly
where s is large, and later steps bring that together.)  Up to five steps 2^-8 = 3.9e-3 is allowed.  Where singular values are near 1, the steps go on mapping them between 0.7 and 1.2 and errors no
longer shrink: 2^-7 is allowed for six to eight."""
import torch

CASES = [("gauss", s) for s in ((130, 200), (256, 256), (512, 512), (384, 1000), (1000, 384))] + [("low rank", s) for s in ((64, 200), (130, 200), (256, 256), (300, 140), (512, 512), (384, 1000))]
STEPS = (1, 2, 3, 5, 6, 8)


def allowed(steps):
    return 2.0 ** -8 if steps <= 5 else 2.0 ** -7


def gradient(kind, shape):
    gen = torch.Generator().manual_seed(shape[0] * 31 + shape[1])
    g = torch.randn(*shape, generator=gen)
    if kind == "low rank":
        few = max(1, min(shape) // 16)
        g = torch.randn(shape[0], few, generator=gen) @ torch.randn(few, shape[1], generator=gen) + 0.05 * g
    return g * 1e-3

"""The dense operators around the sparse output layer, as measurable cases.

What trains the features that the fixed-fan-in layer reads, and what a user of that layer needs next to it:

  norm       layer norm of the features, forward (``haste_b200.norm.layer_norm_forward``): y = (x - mean) * rstd * weight + bias
             per row, with mean and rstd kept for the backward pass, or without them for inference
  norm_grad  its backward pass (``layer_norm_backward``): the gradient of the input, of the weight and of the bias
  gradnorm   the 2-norm of all gradients of a step (``haste_b200.optim.grad_norm``), what clipping goes by
  adamw      one AdamW step over many tensors (``adamw_step``), moments in 32 bits or in 8, bf16 weights rounded stochastically,
             gradients clipped by their norm or not

Weights, gradients and moments of the tensors lie in one buffer each, every tensor at a multiple of 256 elements.  Moments in 8
bits have a scale for each 256 elements: the first moment a sign, 4 bits of exponent and 3 of mantissa, the second 5 and 3; both are
rounded stochastically (a moment that moves by a thousandth a step would otherwise never leave its code).  The random bits of
elements 4i .. 4i+3 of the buffer are the four words of Philox4x32 with 7 rounds, key (seed, step), counter (i, 0, 0, 1): the lower
16 bits of a word round the weight, the next 8 the first moment, the highest 8 the second.

Sizes are the feature widths and batches of this package's layers (512 to 4096 features, 64 to 1024 rows), token counts of an encoder
in front of them, and stacks of square and wide matrices with an embedding.
"""
import functools
import math
import random

import torch

own = False

EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256          # elements that share a scale, and what a tensor's place in the buffers is a multiple of
TOP = 1.875          # value of the highest code
TINY = 2.0 ** -120   # a block whose largest value is below this holds zeros

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, kind, rows, width, x, w, stats=True):
    c = dict(kind=kind, rows=rows, width=width, x=x, w=w, stats=stats)
    return dict(c, name=name) if name else c


def _adamw(name, kind, bits, w, g, clip, width=0, wide=0, depth=0, vocab=0, count=0, biggest=0):
    c = dict(kind=kind, bits=bits, w=w, g=g, clip=clip, width=width, wide=wide, depth=depth, vocab=vocab, count=count, biggest=biggest)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one query while serving: the features of a single row, no statistics kept; latency is all that counts
        _norm("norm-1x768", "norm", 1, 768, "bf16", "bf16", stats=False),
        # one training batch of pooled features ahead of the output layer, fp32 activations
        _norm("norm-512x768-f32", "norm", 512, 768, "fp32", "fp32"),
        # all tokens of an encoder's batch
        _norm("norm-65536x1024", "norm", 65536, 1024, "bf16", "bf16"),
        # backward of a small batch of pooled features
        _norm("norm-grad-64x768-f32", "norm_grad", 64, 768, "fp32", "fp32"),
        # an odd number of rows of an odd width: no row but the first starts on 16 bytes
        _norm("norm-grad-4099x1021", "norm_grad", 4099, 1021, "bf16", "bf16"),
        # backward over all tokens of a batch at the widest features, weights kept in fp32
        _norm("norm-grad-32768x4096", "norm_grad", 32768, 4096, "bf16", "fp32"),
        # gradients of a small trained head: a projection and its norm
        _adamw("gradnorm-head", "gradnorm", 0, "fp32", "fp32", 0.0, width=512, wide=512, depth=0, vocab=768),
        # gradients of an encoder, bf16
        _adamw("gradnorm-stack-56m", "gradnorm", 0, "bf16", "bf16", 0.0, width=768, wide=2048, depth=6, vocab=30000),
        # the optimizer step of the small head in fp32
        _adamw("adamw-head-f32", "adamw", 32, "fp32", "fp32", 0.0, width=512, wide=512, depth=0, vocab=768),
        # a large encoder: bf16 weights, moments in 32 bits, clipped
        _adamw("adamw-stack-133m", "adamw", 32, "bf16", "bf16", 1.0, width=1024, wide=2048, depth=12, vocab=32000),
        # many small fp32 tensors of odd sizes, moments in 8 bits
        _adamw("adamw8-ragged-f32", "adamw", 8, "fp32", "fp32", 0.0, count=150, biggest=60000),
        # an encoder with moments in 8 bits, bf16 weights, clipped
        _adamw("adamw8-stack-56m", "adamw", 8, "bf16", "bf16", 1.0, width=768, wide=2048, depth=6, vocab=30000),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "gradnorm", "adamw", "adamw"])
    types = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
    if kind in ("norm", "norm_grad"):
        width = rng.choice([512, 768, 1024, 2048, 4096]) if rng.random() < 0.5 else _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, min(65536, 2 ** 26 // width))
        return _norm(None, kind, rows, width, types[0], types[1], stats=kind == "norm_grad" or rng.random() < 0.7)
    bits = 0 if kind == "gradnorm" else rng.choice([8, 32])
    clip = rng.choice([0.0, 1.0]) if kind == "adamw" else 0.0
    w, g = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
    if rng.random() < 0.35:
        return _adamw(None, kind, bits, w, g, clip, count=_log_int(rng, 1, 200), biggest=_log_int(rng, 1, 400000))
    width = rng.choice([256, 384, 512, 768, 1024])
    return _adamw(None, kind, bits, w, g, clip, width=width, wide=rng.choice([2, 3]) * width if width < 1024 else 2 * width, depth=rng.randint(0, 8),
                  vocab=_log_int(rng, 500, 32000))


def _shapes(c):
    """Shapes of the tensors: an embedding, and per layer four square matrices, two wide ones, their biases and two norms; or
    tensors of any sizes."""
    if c["count"]:
        rng = random.Random(c["count"] * 1000003 + c["biggest"])
        return [(_log_int(rng, 1, c["biggest"]),) for _ in range(c["count"])]
    d, f = c["width"], c["wide"]
    layer = [(d, d), (d,)] * 4 + [(f, d), (f,), (d, f), (d,)] + [(d,)] * 4
    return [(c["vocab"], d), (d,), (d,)] + layer * c["depth"]


def _views(flat, shapes):
    """The tensors in their buffer."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += -(-n // BLOCK) * BLOCK
    return out


def _encode(x, signed, rnd):
    """(codes uint8, scales fp32) of a buffer in blocks of 256; rnd: 8 random bits an element (int32), 128 and a half for nearest."""
    top = x.view(-1, BLOCK).abs().amax(1)
    fine = top >= TINY
    scales = torch.where(fine, top * (1.0 / TOP), 0.0)
    y = (x.view(-1, BLOCK) * torch.where(fine, TOP / top, 0.0)[:, None]).view(-1)
    most, base = (127, 0x380) if signed else (255, 0x300)
    code = (((y.abs().view(torch.int32) + (rnd << 12) + 0x800) >> 20) - base).clamp_(0 if signed else 1, most)
    code = torch.where(y == 0, 0, code)
    if signed:
        code = torch.where((y < 0) & (code > 0), code + 128, code)
    return code.to(torch.uint8), scales


def _decode(codes, scales, signed):
    c = codes.to(torch.int32)
    mag = c & 127 if signed else c
    y = torch.where(mag == 0, 0.0, ((mag + (0x380 if signed else 0x300)) << 20).view(torch.float32))
    if signed:
        y = torch.where(c > 127, -y, y)
    return (y.view(-1, BLOCK) * scales[:, None]).view(-1)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = functools.partial(torch.randn, generator=gen, device="cuda")
    if c["kind"] in ("norm", "norm_grad"):
        R, D = c["rows"], c["width"]
        # hidden states: rows of different scale, a few columns that stand out, a mean that is not zero
        x = randn(R, D) * (randn(R, 1) * 0.3).exp_() * (1.0 + 4.0 * (torch.rand(D, generator=gen, device="cuda") < 0.02)) + 0.1 * randn(D)
        x = x.to(_TYPES[c["x"]])
        w = (1.0 + 0.2 * randn(D)).to(_TYPES[c["w"]])
        b = (0.1 * randn(D)).to(_TYPES[c["w"]])
        if c["kind"] == "norm":
            return dict(case=c, x=x, w=w, b=b)
        x32 = x.float()
        mean = x32.mean(1)
        rstd = ((x32 - mean[:, None]).square().mean(1) + EPS).rsqrt()
        return dict(case=c, x=x, w=w, mean=mean, rstd=rstd, dy=(randn(R, D) * 1e-2).to(_TYPES[c["x"]]))
    shapes = _shapes(c)
    mask = torch.cat([torch.arange(-(-math.prod(s) // BLOCK) * BLOCK, device="cuda") < math.prod(s) for s in shapes])
    n = mask.numel()
    # gradients of different size from run to run of 64 elements, a third of the runs untouched (rows of an embedding that no
    # token asked for)
    size = ((randn(n // 64) * 1.0).exp_() * 1e-3).repeat_interleave(64)
    hit = (torch.rand(n // 64, generator=gen, device="cuda") > 0.33).repeat_interleave(64)
    g = (randn(n) * size * hit * mask).to(_TYPES[c["g"]])
    state = dict(case=c, g=g, grads=_views(g, shapes))
    if c["kind"] == "gradnorm":
        return state
    m, v = 0.3 * randn(n) * size * mask, size.square() * (0.5 + torch.rand(n, generator=gen, device="cuda")) * mask
    w = (0.02 * randn(n) * mask).to(_TYPES[c["w"]])
    half = torch.full((n,), 127, dtype=torch.int32, device="cuda")
    state.update(w=w, params=_views(w, shapes), seed=int(seed) & 0x7FFFFFFF, step=1000)
    if c["bits"] == 8:
        state.update(m=_encode(m, True, half), v=_encode(v, False, half))
    else:
        state.update(m=m, v=v)
    return state


# ------------------------------------------------------------------ the framework's operators
@functools.lru_cache(maxsize=None)
def _framework():
    from haste_b200 import norm, optim
    return norm, optim


def _run_own(s):
    c = s["case"]
    norm, optim = _framework()
    if c["kind"] == "norm":
        if not c["stats"]:
            return norm.layer_norm_forward(s["x"], s["w"], s["b"], EPS, stats=False)
        return norm.layer_norm_forward(s["x"], s["w"], s["b"], EPS)
    if c["kind"] == "norm_grad":
        return norm.layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"])
    if c["kind"] == "gradnorm":
        return optim.grad_norm(s["grads"])
    s["step"] += 1
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        m, v = optim.Quantized(*m, signed=True), optim.Quantized(*v, signed=False)
    total = optim.adamw_step(s["params"], s["grads"], m, v, step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                             max_norm=c["clip"] or None, stochastic_rounding=True, seed=s["seed"])
    out = dict(w=s["w"])
    if c["clip"]:
        out["norm"] = total
    # moments in 8 bits are returned as the values they stand for
    out["m"] = optim.dequantize(m, torch.bfloat16) if c["bits"] == 8 else m
    out["v"] = optim.dequantize(v, torch.bfloat16) if c["bits"] == 8 else v
    return out


# ------------------------------------------------------------------ the plain forms
def _philox7(counter, key0, key1):
    """The four words for every counter (int64, below 2^32), as int64."""
    low = 0xFFFFFFFF
    zero = torch.zeros_like(counter)
    a, b, c, d = counter, zero, zero, zero + 1
    k0, k1 = key0 & low, key1 & low
    for _ in range(7):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return a, b, c, d


def _plain_norm(s):
    c, x = s["case"], s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / (d.square().mean(1) + EPS).sqrt()
    y = (d * rstd[:, None] * s["w"].float() + s["b"].float()).to(s["x"].dtype)
    return (y, mean, rstd) if c["stats"] else y


def _plain_norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["w"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(s["x"].dtype), (dy * xhat).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)


def _plain_adamw(s):
    c = s["case"]
    s["step"] += 1
    g = s["g"].float()
    out = dict(w=s["w"])
    if c["clip"]:
        out["norm"] = g.square().sum().sqrt()
        g = g * (c["clip"] / (out["norm"] + 1e-6)).clamp(max=1.0)
    m, v = (_decode(*s["m"], True), _decode(*s["v"], False)) if c["bits"] == 8 else (s["m"], s["v"])
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g.square()
    rate = LR / (1 - BETA1 ** s["step"])
    w = s["w"].float() * (1 - LR * DECAY) - rate * m / (v.sqrt() * (1 / math.sqrt(1 - BETA2 ** s["step"])) + ADAM_EPS)
    if c["bits"] == 8 or c["w"] == "bf16":
        words = _philox7(torch.arange(w.numel() // 4, device=w.device), s["seed"], s["step"])
        bits = torch.stack(words, 1).view(-1)
    if c["w"] == "bf16":
        w = ((w.view(torch.int32) + (bits & 0xFFFF).to(torch.int32)) & -0x10000).view(torch.float32)
    s["w"].copy_(w)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return dict(out, m=s["m"], v=s["v"])
    q, r = _encode(m, True, ((bits >> 16) & 0xFF).to(torch.int32)), _encode(v, False, (bits >> 24).to(torch.int32))
    s["m"][0].copy_(q[0]), s["m"][1].copy_(q[1]), s["v"][0].copy_(r[0]), s["v"][1].copy_(r[1])
    return dict(out, m=_decode(*s["m"], True).to(torch.bfloat16), v=_decode(*s["v"], False).to(torch.bfloat16))


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "norm_grad":
        return _plain_norm_grad(state)
    if kind == "gradnorm":
        return state["g"].float().square().sum().sqrt()
    return _plain_adamw(state)


# ------------------------------------------------------------------ the definition in 64 bits
def _values(signed):
    """What each code stands for, times its block's scale."""
    if signed:
        half = [0.0] + [math.ldexp(1 + (c % 8) / 8, c // 8 - 15) for c in range(1, 128)]
        return torch.tensor(half + [-x for x in half], dtype=torch.float64, device="cuda")
    return torch.tensor([0.0] + [math.ldexp(1 + (c % 8) / 8, c // 8 - 31) for c in range(1, 256)], dtype=torch.float64, device="cuda")


def exact(case, seed):
    """In 64 bits from the formulas; what is rounded stochastically stands unrounded."""
    c, s = case, prepare(case, seed)
    if c["kind"] in ("norm", "norm_grad"):
        x, w = s["x"].double(), s["w"].double()
        if c["kind"] == "norm":
            var, mean = torch.var_mean(x, 1, correction=0)
            y = torch.addcmul(s["b"].double(), (x - mean[:, None]) / (var + EPS).sqrt()[:, None], w)
            return (y, mean, (var + EPS).rsqrt()) if c["stats"] else y
        # dL/dx_j = r (w_j dy_j - (1/D) sum_k w_k dy_k (1 + z_j z_k)), with z the normalised row
        dy, r = s["dy"].double(), s["rstd"].double()[:, None]
        z = (x - s["mean"].double()[:, None]) * r
        h = dy * w
        dx = r * (h - (h.sum(1, keepdim=True) + z * torch.einsum("ij,ij->i", h, z)[:, None]) / c["width"])
        return dx, torch.einsum("ij,ij->j", dy, z), dy.sum(0)
    g = s["g"].double()
    total = torch.linalg.vector_norm(g)
    if c["kind"] == "gradnorm":
        return total
    out = {}
    if c["clip"]:
        out["norm"] = total
        g = g * min(1.0, c["clip"] / (float(total) + 1e-6))
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        m = _values(True)[m[0].long()] * m[1].double().repeat_interleave(BLOCK)
        v = _values(False)[v[0].long()] * v[1].double().repeat_interleave(BLOCK)
    m = torch.lerp(g, m.double(), BETA1)
    v = torch.lerp(g * g, v.double(), BETA2)
    t = s["step"] + 1
    hat_m, hat_v = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    w = s["w"].double()
    w = w - LR * DECAY * w - LR * hat_m / (hat_v.sqrt() + ADAM_EPS)
    return dict(out, w=w, m=m, v=v)


def work(case):
    c = case
    size = {"bf16": 2, "fp32": 4}
    if c["kind"] in ("norm", "norm_grad"):
        n, x, w = c["rows"] * c["width"], size[c["x"]], size[c["w"]]
        if c["kind"] == "norm":
            return dict(bytes=2 * x * n + 2 * w * c["width"] + (8 * c["rows"] if c["stats"] else 0), flops=8 * n)
        return dict(bytes=3 * x * n + 3 * w * c["width"] + 8 * c["rows"], flops=14 * n)
    n = sum(math.prod(s) for s in _shapes(c))
    if c["kind"] == "gradnorm":
        return dict(bytes=size[c["g"]] * n, flops=2 * n)
    # weights and moments read and written, gradients read; moments in 8 bits with their scales, and out once more as values
    moments = 16 if c["bits"] == 32 else 4 + 16 / BLOCK + 4
    return dict(bytes=int((2 * size[c["w"]] + size[c["g"]] + moments) * n), flops=16 * n)

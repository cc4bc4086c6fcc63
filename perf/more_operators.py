"""The operators of an encoder in front of the sparse output layer, as measurable cases.

What makes the features that the fixed-fan-in layer reads, and what trains its matrices:

  embed        token embedding (``haste_b200.embedding.embedding_forward``): y[t] = scale * table[ids[t]]
  embed_grad   its gradient (``embedding_backward``): dense [vocab, D], every row summed over the tokens that asked for it; a padding row
               and rows of no token get zeros
  gated        gated feed-forward block (``haste_b200.feedforward.gated_forward``): y = (act(x Wg^T) * (x Wu^T)) Wd^T, with the two
               projections kept for the backward pass, or without them for inference
  gated_grad   its backward pass (``gated_backward``) from the kept projections (bf16): the gradients of x and of the three weights
  ortho        the nearest orthogonal matrices by Newton-Schulz steps (``haste_b200.optim.orthogonalize``), for a list of matrices:
               X = G / max(|G|, eps), then ``STEPS`` times X <- a X + (b A + c A^2) X with A = X X^T (X transposed where it has more rows than columns)
  muon         a step of the optimizer that goes by them (``muon_step``): momentum, Nesterov's form of it, the above, decay and update of
               the weights, bf16 weights rounded stochastically

The matrices of a ``muon`` case and their momentum lie in one buffer each, every tensor at a multiple of 256 elements.  The random bits of elements
4i .. 4i+3 of the buffer are the lower halves of the four words of Philox4x32 with 7 rounds, key (seed, step), counter (i, 0, 0, 2).

Sizes are the feature widths and batches of this package's layers (512 to 4096 features, 64 to 1024 rows), token counts of an encoder in front of
them, and stacks of square and wide matrices.
"""
import functools
import math
import random

import torch

own = False

A, B, C = 3.4445, -4.7750, 2.0315       # the Newton-Schulz polynomial's coefficients
STEPS, NORM_EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 2e-3, 0.95, 0.1
BLOCK = 256                             # what a tensor's place in the buffers is a multiple of

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _embed(name, kind, tokens, width, vocab, dtype, pad=-1, scale=1.0):
    c = dict(kind=kind, tokens=tokens, width=width, vocab=vocab, dtype=dtype, pad=pad, scale=scale)
    return dict(c, name=name) if name else c


def _gated(name, kind, tokens, width, hidden, out, act, keep=True):
    c = dict(kind=kind, tokens=tokens, width=width, hidden=hidden, out=out, act=act, keep=keep)
    return dict(c, name=name) if name else c


def _muon(name, kind, g, width=0, wide=0, depth=0, count=0, biggest=0, nesterov=True, adjust="match_rms_adamw"):
    c = dict(kind=kind, g=g, width=width, wide=wide, depth=depth, count=count, biggest=biggest, nesterov=nesterov, adjust=adjust)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one short query while serving: latency is all that counts
        _embed("embed-9x768", "embed", 9, 768, 30000, "bf16"),
        # all tokens of an encoder's batch, scaled by the root of the width
        _embed("embed-65536x1024", "embed", 65536, 1024, 32000, "bf16", scale=32.0),
        # an odd number of tokens at an odd width, fp32, with a padding row
        _embed("embed-grad-4099x1021-f32", "embed_grad", 4099, 1021, 5003, "fp32", pad=0),
        # the gradient of a whole batch: frequent tokens come thousands of times
        _embed("embed-grad-65536x1024", "embed_grad", 65536, 1024, 32000, "bf16", pad=0, scale=32.0),
        # one token while serving: the weights are read once
        _gated("gated-1x768", "gated", 1, 768, 2048, 768, "silu", keep=False),
        # all tokens of a batch, training
        _gated("gated-65536x1024", "gated", 65536, 1024, 2048, 1024, "silu"),
        # backward of a small batch at odd sizes
        _gated("gated-grad-333x509", "gated_grad", 333, 509, 1021, 509, "gelu"),
        # backward at the widest features
        _gated("gated-grad-16384x4096", "gated_grad", 16384, 4096, 4096, 4096, "silu"),
        # the matrix of a small trained head
        _muon("ortho-head", "ortho", "fp32", width=512, wide=768, depth=0),
        # the matrices of an encoder
        _muon("ortho-stack-50m", "ortho", "bf16", width=768, wide=2048, depth=9),
        # many small fp32-gradient matrices of odd sizes
        _muon("muon-ragged", "muon", "fp32", count=40, biggest=600),
        # the step of a large encoder's matrices
        _muon("muon-stack-101m", "muon", "bf16", width=1024, wide=2048, depth=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "gated", "gated", "gated_grad", "ortho", "muon"])
    if kind in ("embed", "embed_grad"):
        width = rng.choice([512, 768, 1024, 2048, 4096]) if rng.random() < 0.5 else _log_int(rng, 1, 4096)
        vocab = _log_int(rng, 2, min(250000, 2 ** 24 // width))
        return _embed(None, kind, _log_int(rng, 1, min(131072, 2 ** 25 // width)), width, vocab, rng.choice(["bf16", "bf16", "fp32"]),
                      rng.choice([-1, 0, vocab - 1]), rng.choice([1.0, math.sqrt(width)]))
    if kind in ("gated", "gated_grad"):
        odd = rng.random() < 0.4
        width = _log_int(rng, 16, 1100) if odd else rng.choice([512, 768, 1024, 2048])
        hidden = _log_int(rng, 16, 2100) if odd else rng.choice([1024, 1536, 2048, 2560])
        out = width if rng.random() < 0.7 else rng.choice([width // 2, 512])
        tokens = _log_int(rng, 1, min(65536, 2 ** 36 // (width * hidden)))
        return _gated(None, kind, tokens, width, hidden, out, rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), keep=kind == "gated_grad" or rng.random() < 0.5)
    g = rng.choice(["bf16", "fp32"])
    more = dict(nesterov=rng.random() < 0.7, adjust=rng.choice(["original", "match_rms_adamw"]))
    if rng.random() < 0.4:
        return _muon(None, kind, g, count=_log_int(rng, 1, 60), biggest=_log_int(rng, 2, 1200), **more)
    width = rng.choice([256, 384, 512, 768, 1024])
    return _muon(None, kind, g, width=width, wide=2 * width + 128 * rng.randint(0, 7), depth=rng.randint(0, 8 if width < 1024 else 3), **more)


def _shapes(c):
    """The matrices: a projection, and per layer four square ones and two wide ones; or matrices of any sizes."""
    if c["count"]:
        rng = random.Random(c["count"] * 1000003 + c["biggest"])
        return [(_log_int(rng, 1, c["biggest"]), _log_int(rng, 1, c["biggest"])) for _ in range(c["count"])]
    d, f = c["width"], c["wide"]
    return [(d, f)] + ([(d, d)] * 4 + [(f, d), (d, f)]) * c["depth"]


def _views(flat, shapes):
    """The tensors in their buffer."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += -(-n // BLOCK) * BLOCK
    return out


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = functools.partial(torch.randn, generator=gen, device="cuda")
    if c["kind"] in ("embed", "embed_grad"):
        T, D, V = c["tokens"], c["width"], c["vocab"]
        # words: the r-th most frequent comes about every r-th of the times that the first does
        ids = (torch.exp(torch.rand(T, generator=gen, device="cuda", dtype=torch.float64) * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
        if c["kind"] == "embed":
            return dict(case=c, ids=ids, table=(0.05 * randn(V, D)).to(_TYPES[c["dtype"]]))
        return dict(case=c, ids=ids, dy=(1e-2 * randn(T, D) * (0.5 * randn(T, 1)).exp_()).to(_TYPES[c["dtype"]]))
    if c["kind"] in ("gated", "gated_grad"):
        T, D, F, O = c["tokens"], c["width"], c["hidden"], c["out"]
        bf = torch.bfloat16
        # normalised features with a few columns that stand out
        x = (randn(T, D) * (1.0 + 2.0 * (torch.rand(D, generator=gen, device="cuda") < 0.02))).to(bf)
        s = dict(case=c, x=x, wg=(randn(F, D) * D ** -0.5).to(bf), wu=(randn(F, D) * D ** -0.5).to(bf), wd=(randn(O, F) * F ** -0.5).to(bf))
        if c["kind"] == "gated_grad":
            s.update(dy=(randn(T, O) * 1e-2).to(bf), gate=(x.float() @ s["wg"].float().t()).to(bf), up=(x.float() @ s["wu"].float().t()).to(bf))
        return s
    shapes = _shapes(c)
    n = sum(-(-math.prod(t) // BLOCK) * BLOCK for t in shapes)
    # gradients: a few directions that carry most of the change, and noise over all of them
    g = torch.zeros(n, device="cuda")
    for v in _views(g, shapes):
        few = max(1, min(v.shape) // 16)
        v.copy_(randn(v.shape[0], few) @ randn(few, v.shape[1]) * (few ** -0.5 * 1e-3) + 2e-4 * randn(*v.shape))
    g = g.to(_TYPES[c["g"]])
    state = dict(case=c, g=g, grads=_views(g, shapes))
    if c["kind"] == "ortho":
        return state
    used = torch.zeros(n, device="cuda")
    for v in _views(used, shapes):
        v.fill_(1.0)
    w = (0.02 * randn(n) * used).to(torch.bfloat16)
    state.update(w=w, params=_views(w, shapes), m=(g.float() * 0.7 + 3e-4 * randn(n)) * used, seed=int(seed) & 0x7FFFFFFF, step=1000)
    return state


# ------------------------------------------------------------------ the framework's operators
@functools.lru_cache(maxsize=None)
def _framework():
    from haste_b200 import embedding, feedforward, optim
    return embedding, feedforward, optim


def _run_own(s):
    c = s["case"]
    embedding, feedforward, optim = _framework()
    if c["kind"] == "embed":
        return embedding.embedding_forward(s["ids"], s["table"], c["scale"])
    if c["kind"] == "embed_grad":
        return embedding.embedding_backward(s["dy"], s["ids"], c["vocab"], c["scale"], None if c["pad"] < 0 else c["pad"])
    if c["kind"] == "gated":
        return feedforward.gated_forward(s["x"], s["wg"], s["wu"], s["wd"], c["act"], keep=c["keep"])
    if c["kind"] == "gated_grad":
        return feedforward.gated_backward(s["dy"], s["x"], s["wg"], s["wu"], s["wd"], s["gate"], s["up"], c["act"])
    if c["kind"] == "ortho":
        return optim.orthogonalize(s["grads"], STEPS, (A, B, C), NORM_EPS)
    s["step"] += 1
    optim.muon_step(s["params"], s["grads"], s["m"], step=s["step"], lr=LR, momentum=MOMENTUM, nesterov=c["nesterov"], weight_decay=DECAY, steps=STEPS,
                    coefficients=(A, B, C), eps=NORM_EPS, adjust=c["adjust"], stochastic_rounding=True, seed=s["seed"])
    return dict(w=s["w"], m=s["m"])


# ------------------------------------------------------------------ the plain forms
def _philox7(counter, key0, key1):
    """The four words for every counter (int64, below 2^32), as int64."""
    low = 0xFFFFFFFF
    zero = torch.zeros_like(counter)
    a, b, c, d = counter, zero, zero, zero + 2
    k0, k1 = key0 & low, key1 & low
    for _ in range(7):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return a, b, c, d


def _act(g, kind):
    """(act(g), act'(g)) in g's type."""
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if kind == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    k = math.sqrt(2.0 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * g * g)


def _plain_embed_grad(s):
    c, ids = s["case"], s["ids"]
    dy = s["dy"].float() if c["pad"] < 0 else s["dy"].float() * (ids != c["pad"])[:, None]
    total = torch.zeros(c["vocab"], c["width"], dtype=torch.float64, device=dy.device).index_add_(0, ids, dy.double())
    return (total * c["scale"]).to(s["dy"].dtype)


def _plain_gated(s):
    c, x = s["case"], s["x"].float()
    gate, up = x @ s["wg"].float().t(), x @ s["wu"].float().t()
    y = ((_act(gate, c["act"])[0] * up) @ s["wd"].float().t()).to(torch.bfloat16)
    return (y, gate.to(torch.bfloat16), up.to(torch.bfloat16)) if c["keep"] else y


def _plain_gated_grad(s):
    c, bf = s["case"], torch.bfloat16
    dy, x, gate, up = s["dy"].float(), s["x"].float(), s["gate"].float(), s["up"].float()
    a, slope = _act(gate, c["act"])
    dh = dy @ s["wd"].float()
    dgate, dup = dh * up * slope, dh * a
    dx = dgate @ s["wg"].float() + dup @ s["wu"].float()
    return dx.to(bf), (dgate.t() @ x).to(bf), (dup.t() @ x).to(bf), (dy.t() @ (a * up)).to(bf)


def _newton_schulz(x):
    """The steps for matrices [batch, rows, columns] of one shape, in x's type."""
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    x = x / x.double().square().sum((1, 2), keepdim=True).sqrt().clamp(min=NORM_EPS).to(x.dtype)
    for _ in range(STEPS):
        a = x @ x.transpose(1, 2)
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.transpose(1, 2) if tall else x


def _orthogonal(matrices):
    """The steps for each of a list, matrices of one shape at once."""
    out = [None] * len(matrices)
    for shape in sorted({m.shape for m in matrices}):
        at = [i for i, m in enumerate(matrices) if m.shape == shape]
        for i, o in zip(at, _newton_schulz(torch.stack([matrices[i] for i in at]))):
            out[i] = o
    return out


def _rate(shape, adjust):
    rows, columns = shape
    return 0.2 * math.sqrt(max(rows, columns)) if adjust == "match_rms_adamw" else math.sqrt(max(1.0, rows / columns))


def _plain_muon(s):
    c = s["case"]
    s["step"] += 1
    shapes, g = _shapes(c), s["g"].float()
    m = MOMENTUM * s["m"] + (1 - MOMENTUM) * g
    u = MOMENTUM * m + (1 - MOMENTUM) * g if c["nesterov"] else m
    w = s["w"].float() * (1 - LR * DECAY)
    for v, o in zip(_views(w, shapes), _orthogonal(_views(u, shapes))):
        v.sub_(o, alpha=LR * _rate(v.shape, c["adjust"]))
    bits = torch.stack(_philox7(torch.arange(w.numel() // 4, device=w.device), s["seed"], s["step"]), 1).view(-1)
    s["w"].copy_(((w.view(torch.int32) + (bits & 0xFFFF).to(torch.int32)) & -0x10000).view(torch.float32))
    s["m"].copy_(m)
    return dict(w=s["w"], m=s["m"])


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "embed":
        return (state["table"][state["ids"]].float() * state["case"]["scale"]).to(state["table"].dtype)
    if kind == "embed_grad":
        return _plain_embed_grad(state)
    if kind == "gated":
        return _plain_gated(state)
    if kind == "gated_grad":
        return _plain_gated_grad(state)
    if kind == "ortho":
        return [o.to(torch.bfloat16) for o in _orthogonal([g.float() for g in state["grads"]])]
    return _plain_muon(state)


# ------------------------------------------------------------------ the definition in 64 bits
def _value_and_slope(g, kind):
    """act and its derivative from the definitions, in 64 bits."""
    g = g.detach().requires_grad_(True)
    with torch.enable_grad():
        if kind == "silu":
            y = g * torch.sigmoid(g)
        elif kind == "relu":
            y = torch.clamp(g, min=0.0)
        elif kind == "gelu":
            y = g * torch.special.ndtr(g)
        else:
            y = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        slope, = torch.autograd.grad(y.sum(), g)
    return y.detach(), slope


def _exact_orthogonal(g):
    """p(G): the steps as polynomials of the Gram matrix of G, which commutes with its own powers: X_k = G q_k(G^T G), smaller side out."""
    g = g.double()
    tall = g.shape[0] > g.shape[1]
    x = (g.t() if tall else g) / max(float(torch.linalg.matrix_norm(g)), NORM_EPS)
    gram = x @ x.t()
    eye = torch.eye(gram.shape[0], dtype=torch.float64, device=g.device)
    factor = eye                                    # X_k = factor x, and X_k X_k^T = factor gram factor
    for _ in range(STEPS):
        a = factor @ gram @ factor
        factor = torch.addmm(A * eye, a, torch.addmm(B * eye, a, eye, alpha=C)) @ factor
    x = factor @ x
    return x.t() if tall else x


def exact(case, seed):
    """In 64 bits from the formulas; what is rounded stochastically stands unrounded."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "embed":
        return torch.index_select(s["table"], 0, s["ids"]).double() * c["scale"]
    if c["kind"] == "embed_grad":
        order = torch.argsort(s["ids"], stable=True)
        sums = torch.cat([torch.zeros(1, c["width"], dtype=torch.float64, device="cuda"), s["dy"][order].double().cumsum(0)])
        ends = torch.searchsorted(s["ids"][order], torch.arange(c["vocab"] + 1, device="cuda"))
        total = (sums[ends[1:]] - sums[ends[:-1]]) * c["scale"]
        if c["pad"] >= 0:
            total[c["pad"]] = 0
        return total
    if c["kind"] in ("gated", "gated_grad"):
        x, wg, wu, wd = (s[k].double() for k in ("x", "wg", "wu", "wd"))
        if c["kind"] == "gated":
            gate, up = torch.einsum("td,fd->tf", x, wg), torch.einsum("td,fd->tf", x, wu)
            y = torch.einsum("tf,of->to", _value_and_slope(gate, c["act"])[0] * up, wd)
            return (y, gate, up) if c["keep"] else y
        dy, up = s["dy"].double(), s["up"].double()
        a, slope = _value_and_slope(s["gate"].double(), c["act"])
        dh = torch.einsum("to,of->tf", dy, wd)
        dgate, dup = dh * up * slope, dh * a
        dx = torch.cat([dgate, dup], 1) @ torch.cat([wg, wu], 0)
        return dx, torch.einsum("tf,td->fd", dgate, x), torch.einsum("tf,td->fd", dup, x), torch.einsum("to,tf->of", dy, a * up)
    if c["kind"] == "ortho":
        return [_exact_orthogonal(g) for g in s["grads"]]
    shapes, g = _shapes(c), s["g"].double()
    m = torch.lerp(g, s["m"].double(), MOMENTUM)
    u = torch.lerp(g, m, MOMENTUM) if c["nesterov"] else m
    w = s["w"].double() - LR * DECAY * s["w"].double()
    for v, x in zip(_views(w, shapes), _views(u, shapes)):
        v -= LR * _rate(v.shape, c["adjust"]) * _exact_orthogonal(x)
    return dict(w=w, m=m)


def work(case):
    c = case
    size = {"bf16": 2, "fp32": 4}
    if c["kind"] in ("embed", "embed_grad"):
        T, D, V, e = c["tokens"], c["width"], c["vocab"], size[c["dtype"]]
        # a table's rows are read as often as different ones are asked for: word r is among T draws with probability 1 - (1 - p_r)^T,
        # p_r = log((r + 2) / (r + 1)) / log(V + 1)
        r = torch.arange(V, dtype=torch.float64)
        p = torch.log((r + 2) / (r + 1)) / math.log(V + 1)
        rows = float((1 - torch.exp(T * torch.log1p(-p.clamp(max=1 - 1e-12)))).sum())
        if c["kind"] == "embed":
            return dict(bytes=int(8 * T + e * D * (rows + T)), flops=T * D)
        return dict(bytes=8 * T + e * D * (T + V), flops=T * D)
    if c["kind"] in ("gated", "gated_grad"):
        T, D, F, O = c["tokens"], c["width"], c["hidden"], c["out"]
        weights = 2 * (2 * D * F + O * F)
        if c["kind"] == "gated":
            return dict(bytes=2 * T * (D + O + (2 * F if c["keep"] else 0)) + weights, flops=2 * T * F * (2 * D + O))
        return dict(bytes=2 * T * (2 * D + O + 2 * F) + 2 * weights, flops=2 * T * F * (4 * D + 2 * O))
    n = flops = 0
    for s in _shapes(c):
        p, q = min(s), max(s)
        n += p * q
        # A and A^2 are symmetric: half of each
        flops += STEPS * (p * p * q + p * p * p + 2 * p * p * q)
    if c["kind"] == "ortho":
        return dict(bytes=(size[c["g"]] + 2) * n, flops=flops)
    return dict(bytes=(size[c["g"]] + 4 + 8) * n, flops=flops)

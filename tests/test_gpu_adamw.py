"""AdamW, gradient norm and 8-bit moments against the 64-bit oracle: values within bounds that follow from fp32 arithmetic, stochastic
roundings and codes against the very random bits they are defined by (oracle/dense_oracle.py)."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do

BF, F32 = torch.bfloat16, torch.float32
SIZES = [1, 255, 256, 257, 0, 768, 4097, 5, 70000, 8, 31]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)


def _flat(tensors, dtype=F32):
    """Tensors in the layout of the moments, on the CPU."""
    out = []
    for t in tensors:
        n = t.numel()
        out.append(torch.cat([t.detach().reshape(-1).cpu().to(dtype), torch.zeros(-n % 256, dtype=dtype)]))
    return torch.cat(out) if out else torch.zeros(0, dtype=dtype)


def _make(sizes, p_type, g_type, bits, seed=0, offset=0):
    """Parameters and gradients (`offset` elements off their allocations' start), random moments in the wanted form."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def tensor(n, dtype, scale):
        t = torch.empty(n + offset, dtype=dtype, device="cuda")
        t[offset:] = (torch.randn(n, generator=gen, device="cuda") * scale * (torch.randn(n, generator=gen, device="cuda")).exp()).to(dtype)
        return t[offset:]

    params, grads = [tensor(n, p_type, 0.05) for n in sizes], [tensor(n, g_type, 1e-3) for n in sizes]
    for g in grads:
        g[torch.rand(g.shape, generator=gen, device="cuda") < 0.2] = 0
    m, v = _flat([tensor(n, F32, 1e-3) for n in sizes]).cuda(), _flat([tensor(n, F32, 1e-3).square() for n in sizes]).cuda()
    if bits == 32:
        return params, grads, m, v
    from haste_b200 import optim
    return params, grads, optim.quantize(m, True), optim.quantize(v, False)


def _values(moment):
    if isinstance(moment, torch.Tensor):
        return moment.cpu().double()
    return do.decode(moment.codes.cpu(), moment.scales.cpu(), moment.signed)


def _check_step(before, after, step, seed, sr, scale=1.0, stream=0, hyper=HYPER):
    """before, after: (params, grads, m, v) as lists / moments, cloned around one step."""
    params, grads, m, v = before
    w, g = _flat(params, torch.float64), _flat(grads, torch.float64)
    (b1, b2), n = hyper["betas"], _flat(params).numel()
    (w1, m1, v1), (tw, tm, tv) = do.adamw(w, g, _values(m), _values(v), step, hyper["lr"], b1, b2, hyper["eps"], hyper["weight_decay"], scale)
    real = _flat([torch.ones(p.numel()) for p in params]).bool()
    words = torch.from_numpy(do.random_words(n, seed, step, stream).astype("int64"))
    got_w = _flat(after[0], torch.float64)
    if params[0].dtype == BF:
        bad = do.check_bf16(got_w[real], w1[real], tw[real], (words & 0xFFFF)[real] if sr else None, "w")
    else:
        bad = do.outside(got_w[real].float(), w1[real], tw[real], "w")
    assert bad is None, bad
    for name, x, t, moment, r8 in (("m", m1, tm, after[2], (words >> 16) & 0xFF), ("v", v1, tv, after[3], words >> 24)):
        x, t = x * real, t * real                                          # padding counts for nothing
        if isinstance(moment, torch.Tensor):
            bad = do.outside(moment.cpu()[real], x[real], t[real], name)
        else:
            bad = do.check_codes(moment.codes.cpu(), moment.scales.cpu(), x, t, r8, moment.signed, name)
        assert bad is None, bad


def _clone(x):
    return x.clone() if isinstance(x, torch.Tensor) else type(x)(x.codes.clone(), x.scales.clone(), x.signed) if hasattr(x, "codes") else [_clone(t) for t in x]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
def test_steps(types, bits, offset):
    from haste_b200 import optim
    state = _make(SIZES, *types, bits, seed=bits + offset, offset=offset)
    for step, seed, sr in ((1, 5, True), (2, 2 ** 32 - 1, False), (1000, 7, True), (3000000, 7, True)):
        before = _clone(state)
        assert optim.adamw_step(*state, step=step, seed=seed, stochastic_rounding=sr, **HYPER) is None
        _check_step(before, state, step, seed, sr)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [113, 1025, 2500])
def test_many_tensors(count, bits):
    """More tensors than the small and the large launch hold."""
    from haste_b200 import optim
    state = _make([(i * 37) % 700 for i in range(count)], BF, BF, bits, seed=count)
    before = _clone(state)
    norm = optim.adamw_step(*state, step=12, seed=3, stream_index=9, max_norm=1e9, **HYPER)
    _check_step(before, state, 12, 3, True, stream=9)
    want = math.sqrt(float(_flat(before[1], torch.float64).square().sum()))
    assert abs(float(norm) - want) <= 1e-6 * want


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_and_gradient_scale(bits):
    from haste_b200 import optim
    state = _make(SIZES, BF, F32, bits)
    for grad_scale, part in ((1.0, 0.25), (0.125, 0.5), (-2.0, 3.0)):
        before = _clone(state)
        total = math.sqrt(float(_flat(before[1], torch.float64).square().sum())) * abs(grad_scale)
        norm = optim.adamw_step(*state, step=4, seed=3, grad_scale=grad_scale, max_norm=part * total, **HYPER)
        assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - total) <= 1e-6 * total
        _check_step(before, state, 4, 3, True, scale=grad_scale * min(1.0, part * total / (float(norm) + 1e-6)))


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_missing_or_zero(bits):
    from haste_b200 import optim
    state = _make(SIZES, BF, BF, bits)
    grads = [None if i in (1, 6) else g for i, g in enumerate(state[1])]
    before = _clone(state)
    optim.adamw_step(state[0], grads, *state[2:], step=4, seed=3, **HYPER)
    at = optim.moment_offsets(SIZES)
    assert at[0] == 0 and at[3] == 768 and all(a % 256 == 0 for a in at)
    full = _clone(before)
    optim.adamw_step(*full, step=4, seed=3, **HYPER)
    for i in range(len(SIZES)):
        same = before if i in (1, 6) else full
        assert torch.equal(state[0][i], same[0][i])
        part = slice(at[i], at[i + 1])
        for k in (2, 3):
            assert torch.equal(_values(state[k])[part], _values(same[k])[part])
    optim.adamw_step(state[0], [None] * len(SIZES), *state[2:], step=5, **HYPER)
    optim.adamw_step([], [], *state[2:], step=5, **HYPER)
    # from zero moments, zero gradients: decay alone
    p = [torch.ones(300, device="cuda")]
    zero = [torch.zeros(512, device="cuda") for _ in range(2)]
    zero = zero if bits == 32 else [optim.quantize(z, s) for z, s in zip(zero, (True, False))]
    optim.adamw_step(p, [torch.zeros(300, device="cuda")], *zero, step=1, **HYPER)
    assert torch.equal(p[0], torch.full((300,), 1 - 3e-3 * 0.02, device="cuda")) and not any(bool(_values(z).any()) for z in zero)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_gradients_that_are_not_finite(value, bits):
    from haste_b200 import optim
    state = _make([700, 300], BF, F32, bits)
    state[1][0][400] = value
    before = _clone(state)
    norm = optim.adamw_step(*state, step=4, max_norm=1.0, **HYPER)
    assert not math.isfinite(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(before[0], state[0])) and torch.equal(_values(before[2]), _values(state[2])) and torch.equal(_values(before[3]), _values(state[3]))
    # not clipped: its own weight, and in 8 bits its block of 256 moments
    optim.adamw_step(*state, step=4, seed=3, **HYPER)
    w = state[0][0].float()
    assert bool(w[400].isnan())
    m = _values(state[2])
    if bits == 8:
        assert bool(m[256:512].isnan().all()) and not bool(m[:256].isnan().any() | m[512:].isnan().any())
        assert not bool(w[:400].isnan().any() | w[401:].isnan().any())
    else:
        assert not bool(m[:400].isnan().any() | m[401:].isnan().any())
    clean = _clone(before)
    clean[1][0][400] = 0
    optim.adamw_step(*clean, step=4, seed=3, **HYPER)
    others = torch.arange(700) != 400
    assert torch.equal(w.cpu()[others], clean[0][0].float().cpu()[others]) and torch.equal(state[0][1], clean[0][1])


@pytest.mark.parametrize("signed", [True, False])
def test_codes(signed):
    """Every code survives a round trip; values to the nearest code; blocks of zeros, of tiny and of huge values."""
    from haste_b200 import optim
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(5)
    if signed:
        codes[codes == 128] = 0                                            # minus zero is not written
    scales = torch.tensor([1.0, 3e-20, 7e20, 0.37, 0.0], device="cuda")
    values = optim.dequantize(optim.Quantized(codes, scales, signed))
    want = do.decode(codes.cpu(), scales.cpu(), signed)
    assert torch.equal(values.cpu(), want.float())
    assert torch.equal(optim.dequantize(optim.Quantized(codes, scales, signed), BF).cpu(), want.float().bfloat16())
    back = optim.quantize(values, signed)
    assert torch.equal(back.codes[:-256], codes[:-256]) and not back.codes[-256:].any()
    assert torch.allclose(back.scales, scales, rtol=1e-6, atol=0)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(64 * 256, generator=gen, device="cuda") * (torch.randn(64, generator=gen, device="cuda") * 8).exp().repeat_interleave(256)
    x = x if signed else x.square()
    x[:256] = 0
    x[256:512] *= 1e-38 / x[256:512].abs().max()
    x[512:768] *= 3e38 / x[512:768].abs().max()
    q = optim.quantize(x, signed)
    assert do.check_codes(q.codes.cpu(), q.scales.cpu(), x.cpu().double(), 2e-45 + 0 * x.cpu().double(), torch.full((x.numel(),), 127), signed) is None
    assert not q.codes[:512].any() and not q.scales[:2].any()
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[1000] = bad
        z = optim.dequantize(optim.quantize(y, signed))
        assert bool(z[768:1024].isnan().all()) and torch.equal(z[:768], optim.dequantize(q)[:768]) and torch.equal(z[1024:], optim.dequantize(q)[1024:])


def test_stochastic_rounding_is_right_on_average():
    """The mean over 400 seeds of what one step leaves is the value itself within 6 standard errors of a rounding to random bits (whose
    spread is at most half the distance of the two neighbours), and the 2^-9 (8 random bits) or 2^-17 (16) of that distance that the
    last random place may leave."""
    from haste_b200 import optim
    params, grads, m, v = _make([2048], BF, F32, 8)
    n, total = 400, [torch.zeros(2048, dtype=torch.float64, device="cuda") for _ in range(3)]
    for seed in range(n):
        p, mm, vv = _clone(params), _clone(m), _clone(v)
        optim.adamw_step(p, grads, mm, vv, step=50, seed=seed, **HYPER)
        for t, x in zip(total, (p[0].double(), optim.dequantize(mm).double(), optim.dequantize(vv).double())):
            t += x
    (w1, m1, v1), _ = do.adamw(params[0].cpu(), grads[0].cpu(), _values(m), _values(v), 50, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
    for t, x, gap, place in ((total[0], w1, 2.0 ** -7, 2.0 ** -16), (total[1], m1, 2.0 ** -3, 2.0 ** -8), (total[2], v1, 2.0 ** -3, 2.0 ** -8)):
        mean, x = t.cpu() / n, x.float().double()
        allow = gap * x.abs() * (6 * 0.5 / math.sqrt(n) + place) + 1e-6 * x.abs()
        small = x.abs() < x.abs().view(-1, 256).amax(1).repeat_interleave(256) * 2.0 ** -13       # near the first moment's lowest code
        assert bool(((mean - x).abs() <= allow)[~small].all())


def test_moments_in_8_bits_follow_the_gradients():
    """Gradients whose scale changes 20-fold, each element its own way: after 3000 steps the root of the second moment has to be near that of
    fp32 (rounded to nearest, it stays near the old scale for most elements: a spread of 0.6 and more)."""
    from haste_b200 import optim
    n = 8192
    gen = torch.Generator(device="cuda").manual_seed(1)
    a, b = (torch.exp(torch.randn(n, generator=gen, device="cuda") * 1.0) for _ in range(2))
    forms = {bits: [[torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda") for _ in range(2)]] for bits in (32, 8)}
    forms[8][1] = [optim.quantize(z, s) for z, s in zip(forms[8][1], (True, False))]
    for t in range(1, 3001):
        f = min(1.0, t / 1500)
        g = [a ** (1 - f) * b ** f * torch.randn(n, generator=gen, device="cuda")]
        for p, mv in forms.values():
            optim.adamw_step(p, g, *mv, step=t, lr=1e-3, seed=11)
    off = (optim.dequantize(forms[8][1][1]).sqrt() / forms[32][1][1].sqrt()).log()
    assert abs(float(off.mean())) < 0.1 and float(off.std()) < 0.3
    travelled = [float(p[0].double().norm()) for p, _ in forms.values()]
    assert abs(travelled[1] / travelled[0] - 1) < 0.1


def test_gradient_norm():
    from haste_b200 import optim
    gen = torch.Generator(device="cuda").manual_seed(0)
    for sizes in ([1], [0, 3], [5, 256, 1000003], [7] * 1500):
        grads = [torch.randn(n + 1, generator=gen, device="cuda").to((BF, F32)[i % 2])[i % 2:n + i % 2] for i, n in enumerate(sizes)]
        want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        got = optim.grad_norm(grads + [None])
        assert abs(float(got) - want) <= 1e-6 * want and torch.equal(got, optim.grad_norm(grads))
        assert abs(float(optim.grad_norm(grads, -0.5)) - want / 2) <= 1e-6 * want
    assert float(optim.grad_norm([torch.zeros(3, device="cuda")])) == 0.0 and float(optim.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    assert math.isnan(float(optim.grad_norm([torch.tensor([1.0, float("nan")], device="cuda")])))
    assert math.isinf(float(optim.grad_norm([torch.tensor([1.0, float("-inf")], device="cuda", dtype=BF)])))


def test_tensor_of_more_than_2_31_elements():
    """The ends of a tensor beyond 2^31 elements, and a tensor whose moments lie beyond them."""
    from haste_b200 import optim
    n = 2 ** 31 + 300
    sizes = [n, 1000]
    at = optim.moment_offsets(sizes)
    p = [torch.zeros(n, device="cuda", dtype=BF), torch.zeros(1000, device="cuda", dtype=BF)]
    g = [torch.zeros(n, device="cuda", dtype=BF), torch.zeros(1000, device="cuda", dtype=BF)]
    for t in (p[0][:2048], p[0][-2048:], p[1], g[0][:2048], g[0][-2048:], g[1]):
        t.normal_()
    m, v = (optim.Quantized(torch.zeros(at[-1], dtype=torch.uint8, device="cuda"), torch.zeros(at[-1] // 256, device="cuda"), s) for s in (True, False))
    first = (at[1] - 1024) // 256 * 256                                    # of the last blocks of tensor 0
    parts = [(slice(0, 2048), p[0][:2048], g[0][:2048]), (slice(first, at[1]), p[0][first:], g[0][first:]), (slice(at[1], at[2]), p[1], g[1])]
    before = [([a.clone()], [b.clone()], _clone(_part(m, s)), _clone(_part(v, s))) for s, a, b in parts]
    norm = optim.adamw_step(p, g, m, v, step=1, seed=3, max_norm=1e9, **HYPER)
    want = math.sqrt(sum(float(x.double().square().sum()) for x in (g[0][:2048], g[0][-2048:], g[1])))
    assert abs(float(norm) - want) <= 1e-6 * want
    for (s, a, b), old in zip(parts, before):
        words = torch.from_numpy(do.random_words(s.stop - s.start, 3, 1, first=s.start).astype("int64"))
        w, gg = _flat(old[0], torch.float64), _flat(old[1], torch.float64)
        real = _flat([torch.ones(a.numel())]).bool()
        (w1, m1, v1), (tw, tm, tv) = do.adamw(w, gg, 0 * w, 0 * w, 1, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
        assert do.check_bf16(_flat([a], torch.float64)[real], w1[real], tw[real], (words & 0xFFFF)[real]) is None
        for x, t, q, r in ((m1, tm, _part(m, s), (words >> 16) & 0xFF), (v1, tv, _part(v, s), words >> 24)):
            bad = do.check_codes(q.codes.cpu(), q.scales.cpu(), x, t, r, q.signed)
            assert bad is None, bad


def _part(q, s):
    return type(q)(q.codes[s], q.scales[s.start // 256:s.stop // 256], q.signed)


# ------------------------------------------------------------------ the optimizer
def _model(dtype=F32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 64), torch.nn.LayerNorm(64), torch.nn.Linear(64, 7)).cuda().to(dtype)


def _train(model, opt, steps, seed=0, clip=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for _ in range(steps):
        x, y = torch.randn(32, 40, generator=gen, device="cuda"), torch.randn(32, 7, generator=gen, device="cuda")
        opt.zero_grad()
        (model(x.to(next(model.parameters()).dtype)).float() - y).square().mean().backward()
        if clip:
            torch.nn.utils.clip_grad_norm_(model.parameters(), clip)
        opt.step()


@pytest.mark.parametrize("clip", [None, 0.3])
def test_optimizer_follows_torch_in_fp32(clip):
    """Over 20 steps the two differ by rounding alone: each step leaves a relative error of a few ulp in updates of lr, so 20 lr 1e-4 is ample
    (the gradients' own differences enter through the sign-like update m / sqrt(v))."""
    from haste_b200.optim import AdamW
    a, b = _model(), _model()
    kw = dict(lr=1e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    split = lambda m: [{"params": [p for p in m.parameters() if p.dim() > 1]}, {"params": [p for p in m.parameters() if p.dim() < 2], "weight_decay": 0.0}]
    ours = AdamW(split(a), max_grad_norm=clip, **kw)
    _train(a, ours, 20)
    _train(b, torch.optim.AdamW(split(b), **kw), 20, clip=clip)
    for p, q in zip(a.parameters(), b.parameters()):
        assert float((p - q).abs().max()) <= 20 * 1e-3 * 1e-2
    assert (ours.grad_norm is None) == (clip is None)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dicts(bits):
    """A run that is saved and loaded, copied or pickled half-way goes on with the same bits."""
    import io
    from haste_b200.optim import AdamW
    make = lambda m: AdamW(m.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=9)
    a = _model(BF)
    opt = make(a)
    _train(a, opt, 5)
    assert {k for s in opt.state_dict()["state"].values() for k in s} == {"exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if bits == 8 else set())
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    b, c = copy.deepcopy(a), copy.deepcopy(a)
    loaded = make(b)
    loaded.load_state_dict(torch.load(file))
    c, copied = copy.deepcopy((a, opt))
    _train(a, opt, 5, seed=1)
    _train(b, loaded, 5, seed=1)
    _train(c, copied, 5, seed=1)
    for other, o in ((b, loaded), (c, copied)):
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), other.parameters()))
        for s, t in zip(opt.state_dict()["state"].values(), o.state_dict()["state"].values()):
            assert s.keys() == t.keys() and all(torch.equal(s[k], t[k]) for k in s)


def test_state_of_torch_and_of_other_bits():
    from haste_b200.optim import AdamW, dequantize, Quantized
    a = _model()
    ref = torch.optim.AdamW(a.parameters(), lr=1e-2)
    _train(a, ref, 6)
    b, c = copy.deepcopy(a), copy.deepcopy(a)
    opt = AdamW(b.parameters(), lr=1e-2)
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["step_count"] == 6
    _train(a, ref, 3, seed=1)
    _train(b, opt, 3, seed=1)
    assert all(float((p - q).abs().max()) <= 3e-4 for p, q in zip(a.parameters(), b.parameters()))
    # 32 -> 8 -> 32 bits
    small = AdamW(c.parameters(), lr=1e-2, state_bits=8)
    sd = copy.deepcopy(opt.state_dict())
    for group in sd["param_groups"]:
        group["state_bits"] = 8
    small.load_state_dict(sd)
    _train(c, small, 1, seed=2)
    st = small.state[next(c.parameters())]
    assert st["exp_avg"].dtype == torch.uint8 and small.param_groups[0]["step_count"] == 10
    sd = copy.deepcopy(small.state_dict())
    for group in sd["param_groups"]:
        group["state_bits"] = 32
    big = AdamW(c.parameters(), lr=1e-2)
    big.load_state_dict(sd)
    for p in c.parameters():
        p.grad = None
    next(c.parameters()).grad = torch.zeros_like(next(c.parameters()))
    big.step()
    p = next(c.parameters())
    n = p.numel()
    pad = torch.zeros(-(-n // 256) * 256, dtype=torch.uint8, device="cuda")
    pad[:n] = st["exp_avg"].reshape(-1)
    was = dequantize(Quantized(pad, st["exp_avg_scale"], True))[:n].view(p.shape)
    assert torch.allclose(big.state[p]["exp_avg"], 0.9 * was, rtol=1e-6, atol=0)


def test_optimizer_with_mixed_and_unusual_tensors():
    """bf16 and fp32 parameters in one group, a transposed parameter and gradient, a gradient of another type, one that comes and goes."""
    from haste_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    p = [torch.nn.Parameter(t) for t in (rnd(30, 20).to(BF), rnd(50), rnd(20, 33).t(), rnd(9).to(BF), rnd(4, 4))]
    opt = AdamW(p, lr=1e-2, weight_decay=0.0, max_grad_norm=1e9)
    ref = [q.detach().double().cpu().clone() for q in p]
    mom = [(0 * r, 0 * r) for r in ref]
    for step in range(1, 4):
        for i, q in enumerate(p):
            q.grad = rnd(*q.shape).to(q.dtype)
        p[2].grad = rnd(20, 33).t() if step != 2 else rnd(33, 20)
        if step == 2:
            p[4].grad = None
        opt.step()
        total = math.sqrt(sum(float(q.grad.double().square().sum()) for q in p if q.grad is not None))
        assert abs(float(opt.grad_norm) - total) <= 1e-6 * total
        for i, q in enumerate(p):
            if q.grad is None:
                assert torch.equal(q.detach().double().cpu(), last4)
                continue
            (w, m, v), (tol, tm, tv) = do.adamw(ref[i], q.grad.cpu(), *mom[i], step, 1e-2, 0.9, 0.999, 1e-8, 0.0)
            got = q.detach().double().cpu()
            assert bool(((got - w).abs() <= tol + (2.0 ** -7 * w.abs() if q.dtype == BF else 2.0 ** -23 * w.abs()) + 1e-6 * 1e-2).all()), (step, i)
            ref[i], mom[i] = got, (opt.state[q]["exp_avg"].double().cpu(), opt.state[q]["exp_avg_sq"].double().cpu())
        last4 = p[4].detach().double().cpu().clone()
    with pytest.raises(ValueError):
        AdamW(p, state_bits=16)
    with pytest.raises(ValueError):
        AdamW(p, eps=0.0)
    with pytest.raises(ValueError):
        AdamW(p, max_grad_norm=0.0)
    half = torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.half))
    half.grad = torch.zeros_like(half)
    with pytest.raises(RuntimeError):
        AdamW([half]).step()


def test_on_another_stream_and_in_a_graph():
    from haste_b200 import optim
    state = _make(SIZES, BF, BF, 8)
    want, got = _clone(state), _clone(state)
    n0 = optim.adamw_step(*want, step=3, max_norm=0.5, **HYPER)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        n1 = optim.adamw_step(*got, step=3, max_norm=0.5, **HYPER)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    inside = _clone(state)
    with torch.cuda.graph(g):
        n2 = optim.adamw_step(*inside, step=3, max_norm=0.5, **HYPER)
    assert torch.equal(inside[0][3], state[0][3])
    g.replay()
    torch.cuda.synchronize()
    for other, n in ((got, n1), (inside, n2)):
        assert torch.equal(n, n0) and all(torch.equal(a, b) for a, b in zip(want[0], other[0]))
        assert torch.equal(want[2].codes, other[2].codes) and torch.equal(want[3].codes, other[3].codes) and torch.equal(want[2].scales, other[2].scales)


def test_refusals():
    from haste_b200 import optim
    p, g, m, v = _make([300, 20], F32, F32, 32)
    q8 = _make([300, 20], F32, F32, 8)
    ok = dict(step=1)
    bad = [lambda: optim.adamw_step([p[0].cpu(), p[1]], g, m, v, **ok), lambda: optim.adamw_step(p, [g[0].cpu(), g[1]], m, v, **ok), lambda: optim.adamw_step(p, g[:1], m, v, **ok),
           lambda: optim.adamw_step(p, g, m[:512], v[:512], **ok), lambda: optim.adamw_step(p, g, m, v[:512], **ok), lambda: optim.adamw_step(p, g, m, q8[3], **ok),
           lambda: optim.adamw_step(p, g, q8[3], q8[2], **ok), lambda: optim.adamw_step(p, g, m.to(BF), v.to(BF), **ok), lambda: optim.adamw_step(p, g, m.cpu(), v.cpu(), **ok),
           lambda: optim.adamw_step(p, [g[0], g[1].to(BF)], m, v, **ok), lambda: optim.adamw_step([p[0], p[1].to(BF)], g, m, v, **ok),
           lambda: optim.adamw_step([t.half() for t in p], g, m, v, **ok), lambda: optim.adamw_step(p, [t.half() for t in g], m, v, **ok),
           lambda: optim.adamw_step(p, [g[0].view(3, 100), g[1]], m, v, **ok), lambda: optim.adamw_step([p[0].view(30, 10).t(), p[1]], [g[0].view(10, 30), g[1]], m, v, **ok),
           lambda: optim.adamw_step(p, g, m[1:], v[1:], **ok), lambda: optim.adamw_step(p, g, m, v, step=0), lambda: optim.adamw_step(p, g, m, v, step=1, lr=-1.0),
           lambda: optim.adamw_step(p, g, m, v, step=1, lr=float("nan")), lambda: optim.adamw_step(p, g, m, v, step=1, betas=(0.9, 1.0)),
           lambda: optim.adamw_step(p, g, m, v, step=1, betas=(-0.1, 0.9)), lambda: optim.adamw_step(p, g, m, v, step=1, eps=0.0),
           lambda: optim.adamw_step(p, g, m, v, step=1, max_norm=-1.0), lambda: optim.adamw_step(p, g, m, v, step=1, weight_decay=-1.0),
           lambda: optim.adamw_step(p, g, m, v, step=1, grad_scale=float("inf")), lambda: optim.adamw_step(p, g, m, v, step=1, max_norm=1.0, norm=torch.zeros((), device="cuda", dtype=BF)),
           lambda: optim.adamw_step(p, g, m, v, step=1, max_norm=1.0, norm=torch.zeros(())), lambda: optim.grad_norm([]), lambda: optim.grad_norm([g[0].cpu()]),
           lambda: optim.grad_norm([g[0].half()]), lambda: optim.grad_norm([g[0].view(30, 10).t()]), lambda: optim.quantize(m[:100].clone(), True), lambda: optim.quantize(m.to(BF), True),
           lambda: optim.dequantize(optim.Quantized(q8[2].codes, q8[2].scales[:1], True)), lambda: optim.dequantize(q8[2], torch.half),
           lambda: optim.adamw_step(p, g, optim.Quantized(q8[2].codes, q8[2].scales[:1], True), q8[3], **ok)]
    before = _clone((p, g, m, v))
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was not refused")
    assert all(torch.equal(a, b) for a, b in zip(before[0] + [before[2], before[3]], p + [m, v]))

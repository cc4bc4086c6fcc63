"""The optimizer class beside torch's on the same gradients, so that nothing but the two steps' own roundings differs; and state dicts taken
over as they are, from torch's class and between the two forms of moments."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import dense_oracle as do

U = do.U


def _params(seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(*s, generator=gen, device="cuda") * 0.2) for s in ((64, 40), (64,), (7, 64), (1000,))]


def _gradients(params, gen):
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda") * 0.01


@pytest.mark.parametrize("clip", [None, 0.3])
def test_the_same_gradients(clip):
    """What may differ after n steps, for one weight w: per step 3 roundings on each side of terms of the size of w, 6 U |w|; and of lr m / sqrt(v) what the
    moments' own roundings leave.  With betas (0.8, 0.95) a first moment's error is at most 4 U / 0.2 = 20 U of the largest gradient so far, a second one's 4 U / 0.05
    of itself, its root's half of that, 40 U; the largest gradient is at most 1 / sqrt(0.05) = 4.5 times sqrt(v); root, quotient and their like 8 U more on either
    side: 2 (4.5 (20 + 40 + 8) U) = 612 U.  Clipping adds the norms' difference, at most 140 U of every gradient, to both moments: 4.5 * 280 U."""
    from haste_b200.optim import AdamW
    a, b = _params(), _params()
    kw = dict(lr=1e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    split = lambda p: [{"params": p[:1] + p[2:3]}, {"params": p[1:2] + p[3:], "weight_decay": 0.0}]
    ours, ref = AdamW(split(a), max_grad_norm=clip, **kw), torch.optim.AdamW(split(b), **kw)
    gen = torch.Generator(device="cuda").manual_seed(1)
    largest = [p.detach().abs() for p in a]
    for n in range(1, 21):
        _gradients(a, gen)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        if clip:
            torch.nn.utils.clip_grad_norm_(b, clip)
        ours.step()
        ref.step()
        for k, (p, q) in enumerate(zip(a, b)):
            largest[k] = torch.maximum(largest[k], torch.maximum(p.detach().abs(), q.detach().abs()))
            allow = n * (6 * U * largest[k] + 1e-3 * (612 + (1260 if clip else 0)) * U)
            assert bool(((p - q).detach().abs() <= allow).all()), (n, k, float(((p - q).detach().abs() / allow).max()))


def test_moments_of_torch_in_8_bits():
    """A dict of torch's class, not edited: the 8-bit optimizer stays one, and holds what it was given to the nearest code."""
    from haste_b200.optim import AdamW, quantize
    p = _params()
    ref = torch.optim.AdamW(p, lr=1e-2)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(4):
        _gradients(p, gen)
        ref.step()
    opt = AdamW(p, lr=1.0, state_bits=8, stochastic_rounding=False, seed=5)
    opt.load_state_dict(ref.state_dict())
    group = opt.param_groups[0]
    assert (group["state_bits"], group["stochastic_rounding"], group["seed"], group["lr"], group["step_count"]) == (8, False, 5, 1e-2, 4)
    for q in p[1:]:
        q.grad = None
    opt.step()                                                              # lays the moments out; the others have no gradient
    for q in p[1:]:
        s = opt.state[q]
        assert s["exp_avg"].dtype == s["exp_avg_sq"].dtype == torch.uint8
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            flat = torch.zeros(-(-q.numel() // 256) * 256, device="cuda")
            flat[:q.numel()] = ref.state[q][name].reshape(-1)
            want = quantize(flat, signed)
            assert torch.equal(s[name].reshape(-1), want.codes[:q.numel()]) and torch.equal(s[name + "_scale"], want.scales)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_dict_of_the_other_bits_unedited(bits):
    """The values go along, the form stays; and back again for 8 bits, code for code."""
    from haste_b200.optim import AdamW
    p = _params()
    opt = AdamW(p, state_bits=40 - bits, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(4):
        _gradients(p, gen)
        opt.step()
    other = AdamW(copy.deepcopy(p), state_bits=bits)
    back = AdamW(copy.deepcopy(p), state_bits=40 - bits)
    for o, source in ((other, opt), (back, other)):
        o.load_state_dict(source.state_dict())
        for q in o.param_groups[0]["params"]:
            q.grad = None
        o.param_groups[0]["params"][0].grad = torch.zeros(64, 40, device="cuda")
        o.step()
    assert [o.param_groups[0]["state_bits"] for o in (opt, other, back)] == [40 - bits, bits, 40 - bits]
    for i in (1, 2, 3):
        s, t, r = (o.state[o.param_groups[0]["params"][i]] for o in (opt, other, back))
        assert t["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32) and ("exp_avg_scale" in t) == (bits == 8) == ("exp_avg_scale" not in r)
        if bits == 32:
            assert torch.equal(s["exp_avg"], r["exp_avg"]) and torch.equal(s["exp_avg_sq"], r["exp_avg_sq"])

"""Infinities and NaNs among the weights of the gated block: an infinity times a number is an infinity in every form of the second product, from one row to tiles."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF = torch.bfloat16


def _check(T, D, F, O, act, down, up, seed):
    """With infinities of either sign in `down` places of w_down (and a NaN in one) and in `up` of w_up."""
    from haste_b200.feedforward import gated_forward
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    x, wg, wu, wd = r(T, D), r(F, D) * D ** -0.5, r(F, D) * D ** -0.5, r(O, F) * F ** -0.5
    for w, count in ((wd, down), (wu, up)):
        at = torch.randperm(w.numel(), generator=gen)[:count]
        w.view(-1)[at] = torch.tensor([float("inf"), -float("inf")])[torch.randint(0, 2, (count,), generator=gen)]
    if down:
        wd[0, 0] = float("nan")
    x, wg, wu, wd = (t.to(BF).cuda() for t in (x, wg, wu, wd))
    y = gated_forward(x, wg, wu, wd, act)
    (want, *_), _ = eo.gated(x, wg, wu, wd, act, few=1 << 30)
    inf = want.isinf()
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), inf) and torch.equal(y[inf].double(), want[inf])
    return inf


@pytest.mark.parametrize("sizes", [(64, 128, 96), (77, 131, 33), (512, 1024, 512), (40, 2400, 24)])
@pytest.mark.parametrize("T", [1, 2, 5, 7, 8, 9, 16, 17, 32, 33, 300])
def test_infinite_weights(T, sizes):
    D, F, O = sizes
    assert _check(T, D, F, O, "silu", max(1, O // 4), 0, T * 1000 + D).any()
    assert _check(T, D, F, O, "silu", 0, 1, T * 1000 + D + 1).all()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "relu"])
def test_other_activations(act):
    for T in (1, 8, 16, 40):
        _check(T, 64, 72, 40, act, 10, 2, T)

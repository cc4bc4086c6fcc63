"""AdamW where the second moment is subnormal in fp32 and eps is smaller still: its root counts, in 32 bits of moments."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("g_type", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("p_type", [torch.bfloat16, torch.float32])
def test_subnormal_second_moments(p_type, g_type):
    """From zero moments the first step is lr in the direction of the gradient, whatever its size.  With gradients of 2^-60 the second moment is
    0.001 * 2^-120, which 2^-149 resolves to 2^-19 of itself (a rounding: half of that, and half again in the root), so the step is right to 2^-20 and a
    few ulp.  Weights are zero: nothing else is rounded but bf16 weights, to nearest here."""
    from haste_b200.optim import adamw_step
    n, lr = 1000, 0.25
    sign = torch.where(torch.arange(n, device="cuda") % 3 == 0, -1.0, 1.0)
    p, g = [torch.zeros(n, device="cuda", dtype=p_type)], [(sign * 2.0 ** -60).to(g_type)]
    m, v = torch.zeros(1024, device="cuda"), torch.zeros(1024, device="cuda")
    adamw_step(p, g, m, v, step=1, lr=lr, eps=2.0 ** -100, weight_decay=0.0, stochastic_rounding=False)
    assert 0 < float(v[0]) < 2.0 ** -126
    assert float((p[0].float() + lr * sign).abs().max()) <= lr * (2.0 ** -20 + 16 * 2.0 ** -24 + (2.0 ** -8 if p_type == torch.bfloat16 else 0.0))

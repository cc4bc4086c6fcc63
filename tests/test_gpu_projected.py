"""The dense part in front of the sparse layer, trained together with it: the gradients against autograd in fp32 through the same
logits' gradient, the update against the optimizer alone, and training on a task that it can learn."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import ffi_oracle as fo

BF = torch.bfloat16


def _parts(B, H, P, L, F, G, norm_dtype, bias=True, lr=0.0, dense_lr=1e-3, bits=32, clip=None, loss="bce", seed=3):
    from haste_b200.fused import FusedFFIShard
    from haste_b200.norm import LayerNorm
    from haste_b200.optim import AdamW
    from haste_b200.projected import ProjectedFusedStep
    inp = fo.make_inputs(B, P, L, F, G, 3, 1.1, seed=seed, x_kind="normal", bias_zero=False)
    torch.manual_seed(seed)
    lin = torch.nn.Linear(H, P, bias=bias, device="cuda", dtype=BF)
    norm = LayerNorm(P, bias=bias, device="cuda", dtype=norm_dtype)
    with torch.no_grad():
        norm.weight.normal_(1.0, 0.2)
    shard = FusedFFIShard(inp["loc"].cuda(), inp["W"].cuda(), inp["bias"].cuda(), G, P, loss=loss, lr=lr, seed=1, grad_scale=1.0 / B)
    opt = AdamW([{"params": lin.parameters()}, {"params": norm.parameters(), "weight_decay": 0.0}], lr=dense_lr, state_bits=bits, max_grad_norm=clip)
    h = torch.randn(B, H, device="cuda").to(BF)
    return ProjectedFusedStep(lin, norm, shard, opt), h, inp["targets"].cuda(), inp


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("norm_dtype", [BF, torch.float32])
@pytest.mark.parametrize("shape", [(64, 96, 256, 3000, 32, 32), (37, 200, 768, 128 * 9 + 5, 64, 128)])
def test_gradients(shape, norm_dtype, bias):
    B, H, P, L, F, G = shape
    step, h, targets, inp = _parts(*shape, norm_dtype, bias)
    lin, norm, shard = step.projection, step.norm, step.shard
    dh, loss = step.backward(h, targets)
    # the same in fp32 under autograd, with the roundings of a and x to bf16 in place; the logits' gradient is rounded to bf16 as the step does
    leaves = [t.detach().float().requires_grad_(True) for t in (h, lin.weight, norm.weight) + ((lin.bias, norm.bias) if bias else ())]
    hh, w, nw = leaves[:3]
    lb, nb = leaves[3:] if bias else (None, None)
    a = torch.nn.functional.linear(hh, w, lb)
    a = a + (a.to(BF).float() - a).detach()
    x = torch.nn.functional.layer_norm(a, (P,), nw, nb)
    x = x + (x.to(BF).float() - x).detach()
    cols = torch.arange(L, device="cuda") // G
    z = torch.einsum("blf,lf->bl", x[:, shard.loc.long()[cols]], shard.w.float()) + shard.bias.float()
    z = z + (z.to(BF).float() - z).detach()
    y = torch.zeros(B, L, device="cuda")
    y[targets[:, 0].long(), targets[:, 1].long()] = 1.0
    want = torch.nn.functional.binary_cross_entropy_with_logits(z, y, reduction="sum") / B
    want.backward()
    assert abs(float(loss) - float(want.detach())) <= 2e-3 * float(want.detach())
    got = [dh, lin.weight.grad, norm.weight.grad] + ([lin.bias.grad, norm.bias.grad] if bias else [])
    for name, g, leaf in zip(("dh", "dW", "d norm weight", "db", "d norm bias"), got, leaves):
        assert g.shape == leaf.grad.shape, name
        off = (g.float() - leaf.grad).norm() / leaf.grad.norm()
        # bf16 roundings on the way (logits' gradient, da, the result): each 2^-9 at most in rms
        assert float(off) <= 1e-2, (name, float(off))


def test_step_is_backward_and_update():
    step, h, targets, _ = _parts(64, 96, 256, 3000, 32, 32, torch.float32, lr=0.05, clip=0.01)
    other, _, _, _ = _parts(64, 96, 256, 3000, 32, 32, torch.float32, lr=0.05, clip=0.01)
    dh, loss = step.step(h, targets)
    dh2, loss2 = other.backward(h, targets)
    assert torch.equal(step.shard.w, other.shard.w) and torch.allclose(dh.float(), dh2.float(), rtol=2e-2, atol=1e-3 * float(dh.abs().max()))
    assert abs(float(loss) - float(loss2)) <= 1e-4 * float(loss)
    before = other.projection.weight.detach().clone()
    other.update()
    assert not torch.equal(before, other.projection.weight)
    assert abs(float(other.optimizer.grad_norm) - float(step.optimizer.grad_norm)) <= 1e-2 * float(step.optimizer.grad_norm)
    assert step.step(h, targets, want_loss=False)[1] is None


@pytest.mark.parametrize("bits", [32, 8])
def test_it_learns(bits):
    """16 classes of inputs, each with labels of its own: the loss has to fall to a fifth within 60 steps, with moments in 8 bits as in 32."""
    B, H, P, L, F, G = 256, 64, 256, 2000, 64, 64
    step, _, _, _ = _parts(B, H, P, L, F, G, torch.float32, lr=0.2, dense_lr=3e-3, bits=bits, clip=1.0)
    with torch.no_grad():
        step.shard.bias.fill_(-4.0)
    gen = torch.Generator().manual_seed(0)
    centres, labels = torch.randn(16, H, generator=gen), torch.randint(0, L, (16, 5), generator=gen)
    losses = []
    for _ in range(60):
        c = torch.randint(0, 16, (B,), generator=gen)
        h = (centres[c] + 0.3 * torch.randn(B, H, generator=gen)).to(BF).cuda()
        t = torch.stack([torch.arange(B).repeat_interleave(5), labels[c].reshape(-1)], 1).unique(dim=0).to(torch.int32).cuda()
        _, loss = step.step(h, t)
        losses.append(float(loss))
    assert sum(losses[-5:]) < sum(losses[:5]) / 5, (losses[:5], losses[-5:])


def test_refusals():
    from haste_b200.norm import LayerNorm
    from haste_b200.optim import AdamW
    from haste_b200.projected import ProjectedFusedStep
    step, h, targets, _ = _parts(64, 96, 256, 3000, 32, 32, torch.float32)
    lin, norm, shard, opt = step.projection, step.norm, step.shard, step.optimizer
    for args in ((lin, LayerNorm(128, device="cuda"), shard, opt), (torch.nn.Linear(96, 128, device="cuda", dtype=BF), norm, shard, opt),
                 (torch.nn.Linear(96, 256, device="cuda"), norm, shard, opt), (lin, norm, shard, AdamW(lin.parameters()))):
        with pytest.raises(ValueError):
            ProjectedFusedStep(*args)

"""The optimizer class without a GPU, for tests of what it does with its state: the kernel's place is taken by its 64-bit restatement."""
import pytest
import torch

from oracle import dense_oracle as do


@pytest.fixture
def AdamW(monkeypatch):
    """The class, its step computed by the oracle (fp32 parameters, moments in 32 bits)."""
    from haste_b200 import optim

    def step_of(params, grads, m, v, *, step, lr, betas, eps, weight_decay, **_):
        at = optim.moment_offsets([p.numel() for p in params])
        for p, g, a in zip(params, grads, at):
            if g is not None:
                part = slice(a, a + p.numel())
                w1, m1, v1 = do.adamw(p.reshape(-1), g.reshape(-1), m[part], v[part], step, lr, *betas, eps, weight_decay)[0]
                p.copy_(w1.view(p.shape))
                m[part], v[part] = m1.float(), v1.float()

    monkeypatch.setattr(optim, "adamw_step", step_of)
    return optim.AdamW


def make_params(seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(*s, generator=gen)) for s in ((3, 5), (7,), (300,))]


def take_steps(params, opt, n, seed=1):
    gen = torch.Generator().manual_seed(seed)
    for _ in range(n):
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen).to(p.dtype)
        opt.step()


def assert_same(a, b):
    assert all(torch.equal(p, q) for p, q in zip(a, b))

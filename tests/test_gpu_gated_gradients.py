"""The gradients of the gated module against those of the 64-bit formula: all of a gradient at once, in 2-norm and along the gradient itself, where a missing term cannot hide."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
ACTS = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, gelu_tanh=lambda t: torch.nn.functional.gelu(t, approximate="tanh"), relu=torch.relu)
# dy, the kept gate (which counts up to twice, by act'), the kept up, what goes into the last product (dgate, dup or h) and the gradient itself are rounded: 2^-8 of each at most
ALLOWED = 6 * 2 ** -8


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(20, 48, 80, 32), (5, 40, 56, 24), (300, 77, 131, 65), (257, 128, 256, 128)])
def test_gradients(shape, act):
    from haste_b200.feedforward import GatedFeedForward
    T, D, F, O = shape
    torch.manual_seed(T)
    m = GatedFeedForward(D, F, out=O, activation=act, device="cuda")
    x, w = torch.randn(T, D, device="cuda").to(BF).requires_grad_(), torch.randn(T, O, device="cuda")
    (m(x).float() * w).sum().backward()
    leaves = [x, m.w_gate, m.w_up, m.w_down]
    exact = [p.detach().double().requires_grad_() for p in leaves]
    value = lambda ts: (((ACTS[act](ts[0] @ ts[1].t()) * (ts[0] @ ts[2].t())) @ ts[3].t()) * w.double()).sum()
    value(exact).backward()
    for i, (p, q, name) in enumerate(zip(leaves, exact, "x w_gate w_up w_down".split())):
        size = float(q.grad.norm())
        assert float((p.grad.double() - q.grad).norm()) <= ALLOWED * size, name
        # the difference quotient along the kernel's own gradient is the gradient's size
        d, h = p.grad.double() / float(p.grad.double().norm()), 1e-5
        with torch.no_grad():
            slope = (value([t + h * d if i == j else t for j, t in enumerate(exact)]) - value([t - h * d if i == j else t for j, t in enumerate(exact)])) / (2 * h)
        assert abs(float((p.grad.double() * d).sum()) - float(slope)) <= ALLOWED * size, name


def test_a_wrong_gradient_is_seen():
    """Half a gradient, one of another sign, one without a term: each is further off than what is allowed (in the oracle's place, without a kernel)."""
    torch.manual_seed(0)
    g = torch.randn(80, 48, dtype=torch.float64)
    for wrong in (0.5 * g, -g, torch.randn(80, 48, dtype=torch.float64), torch.where(torch.rand(80, 48) < 0.05, 0.0, g)):
        assert float((wrong - g).norm()) > ALLOWED * float(g.norm())

"""Layer norm has no forward-mode derivative: a tensor with a tangent is refused, as the autograd function refuses it, not answered without one."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(which, grad):
    from haste_b200.norm import layer_norm
    args = [torch.randn(4, 64, device="cuda"), torch.randn(64, device="cuda"), torch.randn(64, device="cuda")]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        want = layer_norm(*args)                                            # no tangent: as ever
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            layer_norm(*args)
        args[which] = forward_ad.unpack_dual(args[which]).primal
        assert torch.equal(layer_norm(*args), want)


def test_the_module_refuses_too():
    from haste_b200.norm import LayerNorm
    m = LayerNorm(64, device="cuda").requires_grad_(False)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(4, 64, device="cuda"), torch.ones(4, 64, device="cuda"))
        with pytest.raises(NotImplementedError):
            m(x)

"""Layer norm and tangents of forward mode without a GPU: the kernel's place is taken by a copy."""
import pytest
import torch
from torch.autograd import forward_ad


def test_a_tangent_is_refused_not_dropped(monkeypatch):
    from haste_b200 import ffi, norm
    monkeypatch.setattr(ffi, "layer_norm_forward", lambda x, w, b, eps, stats=True: x.detach().clone())
    x, w = torch.randn(3, 8), torch.ones(8)
    with forward_ad.dual_level():
        assert torch.equal(norm.layer_norm(x, w, None), x)
        for args in ((forward_ad.make_dual(x, x), w, w), (x, forward_ad.make_dual(w, w), None), (x, None, forward_ad.make_dual(w, w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                norm.layer_norm(*args)
            with pytest.raises(NotImplementedError), torch.no_grad():
                norm.layer_norm(*args)
    assert torch.equal(norm.layer_norm(x, w, w), x)

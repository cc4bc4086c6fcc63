"""The dense operators without a GPU: what the C entry points and the Python functions refuse before any CUDA work, and that the
bounds of the kernels' tests see small mistakes."""
import ctypes

import pytest
import torch

from oracle import dense_oracle as do


def _address():
    buf = ctypes.create_string_buffer(256)
    return buf, ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16


def test_layer_norm_entry_points_refuse():
    from haste_b200 import _lib
    f, g = _lib.lib.haste_layer_norm_forward, _lib.lib.haste_layer_norm_backward
    keep, a = _address()
    bad, unsupported = _lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED
    for args, code, word in [((None, a, a, a, a, a, 1, 4, 4, 1e-5, 0, 0), bad, "NULL"), ((a, a, a, None, a, a, 1, 4, 4, 1e-5, 0, 0), bad, "NULL"),
                             ((a, a, a, a, a, None, 1, 4, 4, 1e-5, 0, 0), bad, "together"), ((a, a, a, a, a, a, -1, 4, 4, 1e-5, 0, 0), bad, "negative"),
                             ((a, a, a, a, a, a, 1, 0, 4, 1e-5, 0, 0), bad, "positive"), ((a, a, a, a, a, a, 1, 4, -4, 1e-5, 0, 0), bad, "strides"),
                             ((a, a, a, a, a, a, 1, 4, 4, -1.0, 0, 0), bad, "eps"), ((a, a, a, a, a, a, 1, 4, 4, float("nan"), 0, 0), bad, "eps"),
                             ((a, a, a, a, a, a, 1, 4, 4, 1e-5, 2, 0), unsupported, "type"), ((a, a, a, a, a, a, 1, 4, 4, 1e-5, 0, -1), unsupported, "type"),
                             ((a, a, a, a, a, a, 1, 2 ** 31, 4, 1e-5, 0, 0), unsupported, "int32")]:
        assert f(*args, None) == code and word in _lib.last_error(), (args, _lib.last_error())
    for k, args in enumerate([(None, a, a, a, a, a, a, a, a, 256, 1, 4, 4, 4, 0, 0, 0), (a, a, a, None, a, a, a, a, a, 256, 1, 4, 4, 4, 0, 0, 0),
                              (a, a, a, a, a, a, a, a, None, 256, 1, 4, 4, 4, 0, 0, 0), (a, a, a, a, a, a, a, a, a, 8, 1, 4, 4, 4, 0, 0, 0),
                              (a, a, a, a, a, a, a, a, a + 4, 256, 1, 4, 4, 4, 0, 0, 0), (a, a, a, a, a, a, a, a, a, 256, 1, 4, -1, 4, 0, 0, 0),
                              (a, a, a, a, a, None, a, a, a, 256, 1, 4, 4, 4, 0, 0, 0)]):
        assert g(*args, None) == bad, k
    assert g(a, a, a, a, a, a, a, a, a, 256, 1, 4, 4, 4, 0, 7, 0, None) == unsupported
    assert _lib.lib.haste_layer_norm_backward_scratch(-1, 4) == 0 and _lib.lib.haste_layer_norm_backward_scratch(4, 0) == 0


def test_layer_norm_refuses_cpu_tensors():
    from haste_b200.norm import LayerNorm, layer_norm, layer_norm_backward
    x = torch.randn(3, 8)
    for call in (lambda: layer_norm(x), lambda: LayerNorm(8)(x), lambda: layer_norm_backward(x, x, None, x[:, 0], x[:, 0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("D", [8, 768])
def test_layer_norm_bounds_see_mistakes(D):
    """A variance over D - 1, an eps left out, a mean taken from the row before, a gradient without one of its means: each is outside."""
    gen = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(*s, generator=gen) for s in ((5, D), (D,), (D,), (5, D)))
    x = x * 0.3
    (y, mean, rstd), (ty, tm, tr) = do.layer_norm(x, w, b, 1e-3)
    exact = lambda r, m=mean: (((x.double() - m[:, None]) * r[:, None]) * w + b).float()
    assert do.outside(exact(rstd), y, ty) is None
    var = rstd ** -2 - 1e-3
    for wrong in (exact((var * D / (D - 1) + 1e-3).rsqrt()), exact(var.rsqrt()), exact(rstd, mean.roll(1))):
        assert do.outside(wrong, y, ty) is not None
    (dx, dw, db), (tx, tw, tb) = do.layer_norm_grad(dy, x, w, mean, rstd)
    assert do.outside(dx.float(), dx, tx) is None
    h, z = (dy * w).double(), (x.double() - mean[:, None]) * rstd[:, None]
    r = rstd[:, None]
    for wrong in (r * (h - h.mean(1, keepdim=True)), r * (h - z * (h * z).mean(1, keepdim=True))):
        assert do.outside(wrong.float(), dx, tx) is not None
    assert do.outside((dw - dy[0].double() * z[0]).float(), dw, tw) is not None
    assert do.outside((db - dy[4].double()).float(), db, tb) is not None

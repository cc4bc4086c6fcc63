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


def test_adamw_entry_points_refuse():
    import array
    from haste_b200 import _lib
    f, keep = _lib.lib.haste_adamw_step, _address()
    a = keep[1]
    ptrs, none, sizes = array.array("Q", [a, a]), array.array("Q", [a, 0]), array.array("q", [100, 200])
    p, n, z = ptrs.buffer_info()[0], none.buffer_info()[0], sizes.buffer_info()[0]
    negative, huge = array.array("q", [100, -1]), array.array("q", [1, 2 ** 38])
    base = dict(params=p, grads=p, sizes=z, count=2, m=a, ms=a, v=a, vs=a, room=512, bits=8, pt=0, gt=0, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, step=1, gs=1.0,
                mn=0.0, norm=None, seed=1, stream=0, flags=0)
    bad, unsupported = _lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED
    for change, code, word in [(dict(count=-1), bad, "count"), (dict(grads=None), bad, "NULL"), (dict(sizes=None), bad, "NULL"), (dict(params=None), bad, "NULL"),
                               (dict(sizes=negative.buffer_info()[0]), bad, "negative"), (dict(sizes=huge.buffer_info()[0]), _lib.ERR_TOO_LARGE, "2^38"),
                               (dict(m=None), bad, "NULL"), (dict(v=a + 4), bad, "aligned"), (dict(ms=None), bad, "NULL"), (dict(room=511), bad, "needed"),
                               (dict(bits=16), unsupported, "bits"), (dict(pt=2), unsupported, "type"), (dict(gt=-1), unsupported, "type"), (dict(lr=-1.0), bad, "lr"),
                               (dict(lr=float("inf")), bad, "lr"), (dict(wd=float("nan")), bad, "weight_decay"), (dict(b1=1.0), bad, "betas"), (dict(b2=-0.1), bad, "betas"),
                               (dict(eps=0.0), bad, "eps"), (dict(step=0), bad, "step"), (dict(gs=float("nan")), bad, "grad_scale"), (dict(norm=a, mn=0.0), bad, "max_norm"),
                               (dict(params=n), bad, "parameter 1")]:
        assert f(*dict(base, **change).values(), None) == code and word in _lib.last_error(), (change, _lib.last_error())
    assert f(*dict(base, count=0, params=None, grads=None, sizes=None, m=None, v=None).values(), None) == _lib.OK
    types, wrong = array.array("i", [0, 1]), array.array("i", [0, 3])
    t, w = types.buffer_info()[0], wrong.buffer_info()[0]
    for args in [(p, t, z, 2, 1.0, None, a), (p, t, z, 2, 1.0, a, None), (p, None, z, 2, 1.0, a, a), (n, t, z, 2, 1.0, a, a), (p, t, z, -2, 1.0, a, a), (p, t, z, 2, float("inf"), a, a)]:
        assert _lib.lib.haste_grad_norm(*args, None) == bad
    assert _lib.lib.haste_grad_norm(p, w, z, 2, 1.0, a, a, None) == unsupported
    for args in [(a, a, a, 100, 1), (a, a, a, -256, 1), (None, a, a, 256, 1), (a, a, None, 256, 1)]:
        assert _lib.lib.haste_quantize_moment(*args, None) == bad
        assert _lib.lib.haste_dequantize_moment(*args, 0, None) == bad
    assert _lib.lib.haste_quantize_moment(a, a + 1, a, 256, 1, None) == bad and _lib.lib.haste_quantize_moment(a + 4, a, a, 256, 1, None) == bad
    assert _lib.lib.haste_dequantize_moment(a + 1, a, a, 256, 1, 0, None) == bad and _lib.lib.haste_dequantize_moment(a, a, a + 2, 256, 1, 0, None) == bad
    assert _lib.lib.haste_dequantize_moment(a, a, a, 256, 1, 5, None) == unsupported
    assert _lib.GRAD_NORM_PARTIALS == 4096


def test_adamw_refuses_cpu_tensors():
    from haste_b200 import optim
    p = [torch.nn.Parameter(torch.randn(8))]
    p[0].grad = torch.randn(8)
    for call in (lambda: optim.AdamW(p).step(), lambda: optim.grad_norm([p[0].grad]), lambda: optim.quantize(torch.zeros(256), True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_moment_offsets():
    from haste_b200.optim import moment_offsets
    assert moment_offsets([1, 256, 257, 0, 5]) == [0, 256, 512, 1024, 1024, 1280] and moment_offsets([]) == [0]


def test_code_tables_and_positions():
    """Codes are ordered, every code lies on a whole position, and the checks see a code that is one off, a wrong sign, a wrong scale."""
    assert do.M_CODES[127] == do.V_CODES[255] == 1.875
    for signed, table in ((True, do.M_CODES[:128]), (False, do.V_CODES)):
        t = torch.tensor(table, dtype=torch.float64)
        assert bool((t[1:] > t[:-1]).all())
        assert torch.equal(do.code_position(t[1:], signed), torch.arange(1, len(table), dtype=torch.float64))
        codes = (torch.randperm(256, generator=torch.Generator().manual_seed(0)) % len(table)).to(torch.uint8)
        codes[0] = len(table) - 1
        scale = torch.tensor([0.3])
        x = do.decode(codes, scale, signed)
        tol, half = 1e-7 * x.abs(), torch.full((256,), 127)
        check = lambda c, s=scale: do.check_codes(c, s, x, tol, half, signed)
        assert check(codes) is None
        for wrong in (codes + (codes < len(table) - 1).to(torch.uint8), codes - (codes > 1).to(torch.uint8)):
            assert check(wrong) is not None
        assert check(codes, scale * 1.001) is not None
        if signed:
            assert check(torch.where(codes > 0, codes + 128, codes)) is not None


def test_adamw_bounds_see_mistakes():
    """No bias correction, coupled weight decay, eps inside the root, a moment of the gradient before clipping: each is outside."""
    gen = torch.Generator().manual_seed(2)
    w, g, m = (torch.randn(512, generator=gen) * s for s in (0.05, 1e-3, 1e-3))
    v = (torch.randn(512, generator=gen) * 1e-3).square() + 1e-9
    step, lr, b1, b2, eps, wd = 10, 1e-3, 0.9, 0.999, 1e-6, 0.1
    (w1, m1, v1), (tw, tm, tv) = do.adamw(w, g, m, v, step, lr, b1, b2, eps, wd)
    assert do.outside(w1.float(), w1, tw) is None and do.outside(m1.float(), m1, tm) is None and do.outside(v1.float(), v1, tv) is None
    coupled = do.adamw(w, g + wd * w, m, v, step, lr, b1, b2, eps, 0.0)[0][0]
    for wrong in (w * (1 - lr * wd) - lr * m1 / (v1.sqrt() + eps), coupled, do.adamw(w, g, m, v, step + 1, lr, b1, b2, eps, wd)[0][0],
                  w * (1 - lr * wd) - lr / (1 - b1 ** step) * m1 / (v1 / (1 - b2 ** step) + eps).sqrt()):
        assert do.outside(wrong.float(), w1, tw) is not None
    assert do.outside(do.adamw(w, 1.001 * g, m, v, step, lr, b1, b2, eps, wd)[0][1].float(), m1, tm) is not None
    words = torch.from_numpy(do.random_words(512, 1, step).astype("int64"))
    right = do.stochastic_bf16(w1, words & 0xFFFF).bfloat16()
    assert do.check_bf16(right, w1, tw, words & 0xFFFF) is None
    for wrong in (w1.bfloat16(), do.stochastic_bf16(w1, words >> 16).bfloat16()):
        assert do.check_bf16(wrong, w1, tw, words & 0xFFFF) is not None


def test_optimizer_refuses_what_it_does_not_do():
    from haste_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(RuntimeError, match="amsgrad or maximize"):
            AdamW([p]).load_state_dict(torch.optim.AdamW([p], **kw).state_dict())
    opt = AdamW([p], lr=0.5)
    opt.load_state_dict(torch.optim.AdamW([p], lr=0.25, weight_decay=0.125).state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["state_bits"] == 32 and opt.param_groups[0]["step_count"] == 0
    opt.step()                                             # no gradients: nothing to do
    assert opt.param_groups[0]["step_count"] == 1
    for kw in (dict(lr=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0)), dict(eps=0.0), dict(state_bits=4), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)


def test_the_extension_refuses_what_is_no_tensor():
    from haste_b200 import ffi
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    from haste_b200.optim import adamw_step, grad_norm
    t = torch.zeros(4)
    for call in (lambda: layer_norm_forward(None, None, None), lambda: layer_norm_forward([1.0], None, None), lambda: layer_norm_backward(t, 3, t, t, t),
                 lambda: grad_norm([t, "t"]), lambda: grad_norm([None, None]), lambda: grad_norm([]), lambda: adamw_step([t], [], t, t, step=1),
                 lambda: adamw_step([t], [3], t, t, step=1), lambda: ffi.dequantize_moment(None, None, True)):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: grad_norm(t[0].item()), lambda: grad_norm([t], "1"), lambda: layer_norm_forward(t, None, None, "eps"), lambda: ffi._dense.grad_norm([t]),
                 lambda: adamw_step([t], [t], t, t, step=1, lr="1")):
        with pytest.raises((TypeError, RuntimeError)):
            call()
    assert adamw_step([t, t], [None, None], t, t, step=1) is None                    # nothing to do

"""What the entry points of embedding, gated feed-forward block and Muon refuse without a GPU, sizes of workspaces, and the oracle against itself."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import encoder_oracle as eo


def _status(call):
    from haste_b200 import _lib
    return call(), _lib.last_error()


def test_c_arguments():
    from haste_b200 import _lib
    lib, A16 = _lib.lib, 4096
    bad, un = _lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED
    i64 = lambda *v: (ctypes.c_int64 * len(v))(*v)
    ptr = lambda *v: (ctypes.c_void_p * len(v))(*v)
    for want, call in (
            (bad, lambda: lib.haste_embedding_forward(None, 8, A16, A16, 5, 8, 10, 8, 1.0, 0, None)),
            (bad, lambda: lib.haste_embedding_forward(A16, 8, A16, A16, -1, 8, 10, 8, 1.0, 0, None)),
            (bad, lambda: lib.haste_embedding_forward(A16, 8, A16, A16, 5, 8, 10, 7, 1.0, 0, None)),
            (un, lambda: lib.haste_embedding_forward(A16, 2, A16, A16, 5, 8, 10, 8, 1.0, 0, None)),
            (un, lambda: lib.haste_embedding_forward(A16, 8, A16, A16, 5, 8, 10, 8, 1.0, 5, None)),
            (bad, lambda: lib.haste_embedding_backward(A16, 8, A16, A16, A16, 10, 5, 8, 10, 8, 1.0, -1, 0, 0, None)),
            (bad, lambda: lib.haste_embedding_backward(A16, 8, A16, A16, A16 + 8, 1 << 40, 5, 8, 10, 8, 1.0, -1, 0, 0, None)),
            (_lib.ERR_TOO_LARGE, lambda: lib.haste_embedding_backward(A16, 8, A16, A16, A16, 1 << 60, 1 << 30, 8, 1 << 30, 8, 1.0, -1, 0, 0, None)),
            (bad, lambda: lib.haste_gated_forward(A16, A16, A16, A16, A16, None, A16, A16, 1 << 40, 20, 8, 8, 8, 8, 8, 0, None)),
            (bad, lambda: lib.haste_gated_forward(A16, A16, A16, A16, A16, A16, A16, A16, 1 << 40, 20, 8, 9, 8, 8, 9, 0, None)),
            (bad, lambda: lib.haste_gated_forward(A16, A16, A16, A16, None, None, A16, A16, 1 << 40, 20, 8, 8, 8, 7, 8, 0, None)),
            (un, lambda: lib.haste_gated_forward(A16, A16, A16, A16, None, None, A16, A16, 1 << 40, 20, 8, 8, 8, 8, 8, 4, None)),
            (bad, lambda: lib.haste_gated_backward(A16, A16, A16, A16, A16, A16, A16, A16, A16, A16, A16, A16, 1 << 40, 20, 8, 8, 8, 7, 8, 8, 8, 0, None)),
            (bad, lambda: lib.haste_muon_step(ptr(A16), ptr(A16), i64(4), i64(4), 1, A16, 255, 0, 0, 0.1, 0.9, 1, 0.0, 0, 5, 1.0, 1.0, 1.0, 1e-7, 1, 0, 0, 0, A16, 1 << 40, None)),
            (bad, lambda: lib.haste_muon_step(ptr(A16), ptr(A16), i64(4), i64(4), 1, A16, 256, 0, 0, 0.1, 0.9, 1, 0.0, 0, 5, 1.0, 1.0, 1.0, 1e-7, 0, 0, 0, 0, A16, 1 << 40, None)),
            (bad, lambda: lib.haste_muon_step(ptr(A16), ptr(A16), i64(4), i64(-4), 1, A16, 256, 0, 0, 0.1, 0.9, 1, 0.0, 0, 5, 1.0, 1.0, 1.0, 1e-7, 1, 0, 0, 0, A16, 1 << 40, None)),
            (un, lambda: lib.haste_muon_step(ptr(A16), ptr(A16), i64(4), i64(4), 1, A16, 256, 0, 0, 0.1, 0.9, 1, 0.0, 2, 5, 1.0, 1.0, 1.0, 1e-7, 1, 0, 0, 0, A16, 1 << 40, None)),
            (bad, lambda: lib.haste_orthogonalize(ptr(A16), ptr(None), i64(4), i64(4), 1, 0, 5, 1.0, 1.0, 1.0, 1e-7, A16, 1 << 40, None)),
            (bad, lambda: lib.haste_orthogonalize(ptr(A16), ptr(A16), i64(4), i64(4), 1, 0, 5, 1.0, 1.0, float("inf"), 1e-7, A16, 1 << 40, None)),
            (bad, lambda: lib.haste_orthogonalize(ptr(A16), ptr(A16), i64(4), i64(4), 1, 0, 5, 1.0, 1.0, 1.0, 1e-7, A16 + 16, 1 << 40, None)),
            (_lib.ERR_TOO_LARGE, lambda: lib.haste_orthogonalize(ptr(A16), ptr(A16), i64(1 << 17), i64(1 << 17), 1, 0, 5, 1.0, 1.0, 1.0, 1e-7, A16, 1 << 60, None))):
        status, why = _status(call)
        assert status == want, why
    # nothing to do
    assert lib.haste_embedding_forward(None, 8, None, None, 0, 8, 10, 8, 1.0, 0, None) == _lib.OK
    assert lib.haste_gated_forward(None, None, None, None, None, None, None, None, 0, 0, 8, 8, 8, 8, 8, 0, None) == _lib.OK
    assert lib.haste_orthogonalize(None, None, None, None, 0, 0, 5, 1.0, 1.0, 1.0, 1e-7, None, 0, None) == _lib.OK


def test_workspaces():
    from haste_b200 import _lib
    lib = _lib.lib
    i64 = lambda v: (ctypes.c_int64 * len(v))(*v)
    assert lib.haste_embedding_backward_scratch(-1, 8, 8) == 0 and lib.haste_gated_forward_scratch(0, 8, 8, 8, 1) == 0
    for T, D, F, O in ((9, 8, 16, 8), (1000, 512, 1024, 256), (70000, 1024, 2048, 1024), (50, 77, 33, 5)):
        fine, any_ = (lib.haste_gated_forward_scratch(T, D, F, O, k) for k in (1, 0))
        assert T * F * 2 <= fine <= any_
        fine, any_ = (lib.haste_gated_backward_scratch(T, D, F, O, k) for k in (1, 0))
        assert 3 * T * F * 2 <= fine <= any_
    one = lib.haste_muon_scratch(i64([1000]), i64([600]), 1)
    assert 6 * 600 * 1000 + 2 * 600 * 600 <= one == lib.haste_muon_scratch(i64([600]), i64([1000]), 1)
    assert lib.haste_muon_scratch(i64([4096] * 100), i64([4096] * 100), 100) <= 1 << 30
    assert lib.haste_muon_scratch(i64([16384]), i64([32768]), 1) > 1 << 30


def test_python_refusals():
    from haste_b200.embedding import Embedding, embedding_backward, embedding_forward
    from haste_b200.feedforward import GatedFeedForward, gated_backward, gated_forward
    from haste_b200.optim import Muon, muon_step, orthogonalize
    x = torch.zeros(4, 8)
    b = x.to(torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: embedding_forward(ids, x), lambda: embedding_backward(x, ids, 4), lambda: embedding_backward(x, ids, 4, 1.0, 9), lambda: gated_forward(b, b, b, b), lambda: gated_forward(b, b, b, b, "tanh"),
                 lambda: gated_backward(b, b, b, b, b, b, b), lambda: muon_step([x], [x], x, step=1), lambda: muon_step([x], [x], x, step=1, adjust="rms"), lambda: orthogonalize([x])):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: Embedding(4, 8, padding_idx=4), lambda: GatedFeedForward(8, 8, activation="tanh"), lambda: Muon([torch.nn.Parameter(x[0])]), lambda: Muon([torch.nn.Parameter(x)], steps=0)):
        with pytest.raises(ValueError):
            call()
    opt = Muon([torch.nn.Parameter(x)])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(x[0])]))
    assert len(opt.param_groups) == 1
    assert set(Embedding(4, 8, padding_idx=-1).state_dict()) == set(torch.nn.Embedding(4, 8).state_dict())


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "relu"])
def test_oracle_of_the_block(kind):
    """The oracle's gradients are those of its forward pass."""
    torch.manual_seed(0)
    f = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, gelu_tanh=lambda t: torch.nn.functional.gelu(t, approximate="tanh"), relu=torch.relu)[kind]
    x, wg, wu, wd = (torch.randn(s, dtype=torch.float64, requires_grad=True) for s in ((6, 5), (7, 5), (7, 5), (4, 7)))
    dy = torch.randn(6, 4, dtype=torch.float64)
    gate, up = x @ wg.t(), x @ wu.t()
    y = (f(gate) * up) @ wd.t()
    (want, *_), _ = eo.gated(*(t.detach() for t in (x, wg, wu, wd)), kind)
    assert torch.allclose(want, y, rtol=1e-10)
    grads = torch.autograd.grad(y, (x, wg, wu, wd), dy)
    got, tol = eo.gated_grad(dy, *(t.detach() for t in (x, wg, wu, wd, gate, up)), kind)
    for a, b, name in zip(got, grads, "x g u d"):
        assert float((a - b).norm()) <= 2 ** -7 * float(b.norm()), name              # the oracle rounds dgate, dup and h


def test_oracle_of_the_steps():
    torch.manual_seed(1)
    g = torch.randn(40, 70, dtype=torch.float64)
    u, s, v = torch.linalg.svd(g / g.norm(), full_matrices=False)
    for _ in range(5):
        s = eo.A * s + eo.B * s ** 3 + eo.C * s ** 5
    assert torch.allclose(eo.orthogonalize(g), u @ torch.diag(s) @ v, atol=1e-10)
    assert torch.allclose(eo.orthogonalize(g.t()), eo.orthogonalize(g).t(), atol=1e-12)
    exact, tol = eo.orthogonalize_bound(g)
    assert 0 < tol < 0.02 * float(exact.norm())


def test_oracle_of_the_embedding():
    torch.manual_seed(2)
    ids, dy = torch.tensor([[1, 3, 1], [0, 9, -1]]), torch.randn(2, 3, 4)
    got, tol = eo.embedding_grad(dy, ids, 5, 2.0, 0)
    want = torch.zeros(5, 4, dtype=torch.float64)
    want[1], want[3] = 2 * (dy[0, 0] + dy[0, 2]).double(), 2 * dy[0, 1].double()
    assert torch.allclose(got, want, atol=1e-6) and (tol >= 0).all() and not got[0].any()
    assert np.isnan(eo.embedding(ids, torch.ones(5, 4), 1.0)[0][1, 1:].numpy()).all()

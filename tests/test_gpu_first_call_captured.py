"""The first call of a process may be one that a CUDA graph captures: each form in a process of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

from conftest import ROOT

CODE = """
import torch
from haste_b200 import ffi
gen = torch.Generator(device="cuda").manual_seed(0)
r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
x, dy = r(300, 64).bfloat16(), r(300, 64).bfloat16()
ws = [r(*s).bfloat16() for s in ((128, 64), (128, 64), (64, 128))]
gate, up, matrix = r(300, 128).bfloat16(), r(300, 128).bfloat16(), r(100, 200)
ids = torch.randint(0, 500, (%(tokens)d,), generator=gen, device="cuda")
grad = r(%(tokens)d, 40)
def call():
    from haste_b200.embedding import embedding_backward, embedding_forward
    from haste_b200.feedforward import gated_backward, gated_forward
    from haste_b200.optim import orthogonalize
    out = %(call)s
    return [out] if isinstance(out, torch.Tensor) else list(out)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
for t in got:
    t.zero_()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, call()))
assert ffi.lib.haste_poll_status() == 0
"""


@pytest.mark.parametrize("call", ["gated_forward(x, *ws, keep=True)", "gated_forward(x[:5], *ws)", "gated_backward(dy, x, *ws, gate, up)", "orthogonalize([matrix, matrix.t().contiguous()])",
                                  "embedding_forward(ids, grad[:500])", "embedding_backward(grad, ids, 500)"])
def test_first_call(call):
    p = subprocess.run([sys.executable, "-c", CODE % dict(call=call, tokens=5000)], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]


def test_first_gradient_of_many_tokens():
    """What sorts them has three forms, whose blocks the device is asked about."""
    p = subprocess.run([sys.executable, "-c", CODE % dict(call="embedding_backward(grad, ids, 500)", tokens=70000)], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True,
                       timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]

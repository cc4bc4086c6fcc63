"""Where the extension of the dense operators does not load (another torch than it was built against, or the library alone), the sparse layer
imports and works as it does without them, and the dense operators say what is missing."""
import subprocess
import sys

from conftest import ROOT

PROGRAM = """
import sys
sys.modules["haste_b200._dense"] = None             # what an extension that does not load comes to
import torch
import haste_b200.fused, haste_b200.shared_ffi, haste_b200.headtail, haste_b200.infer, haste_b200.checkpoint
from haste_b200 import ffi, norm, optim, projected
loc = torch.tensor([[0, 1]], dtype=torch.int32)
try:
    ffi.check_locations(loc, 2)
except RuntimeError as e:
    assert "CUDA" in str(e), e                       # looked at as ever
x = torch.zeros(2, 8)
for call in (lambda: norm.layer_norm(x), lambda: optim.grad_norm([x]), lambda: optim.adamw_step([x], [x], x, x, step=1), lambda: norm.layer_norm_forward(x, None, None)):
    for _ in range(2):
        try:
            call()
        except ImportError as e:
            assert "haste_b200.build" in str(e), e
        else:
            raise AssertionError("not refused")
optim.AdamW([torch.nn.Parameter(x)])                 # nothing is called yet
print("fine")
"""


def test_the_sparse_layer_needs_no_extension():
    p = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True)
    assert p.returncode == 0 and p.stdout.strip() == "fine", p.stderr[-2000:]


def test_the_extension_is_loaded_once():
    from haste_b200 import ffi
    assert ffi._dense.has_tangent(None, None, None) is False
    assert ffi._dense.grad_norm is ffi._dense.__dict__["grad_norm"] and not hasattr(ffi._dense, "no_such_function")

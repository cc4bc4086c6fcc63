"""Gated feed-forward block for an encoder in front of the sparse layer: operator, autograd function and module.

    gated_feed_forward(x, w_gate, w_up, w_down, activation)   under autograd
    GatedFeedForward(features, hidden)                        module
    gated_forward, gated_backward                             the kernels, for steps without an autograd graph

y = (act(x w_gate^T) * (x w_up^T)) w_down^T in bf16, with fp32 sums.
"""
import torch

from . import ffi as _ffi
from ._lib import ACTIVATIONS
from .ffi import gated_backward, gated_forward  # noqa: F401


class _GatedFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        y, gate, up = _ffi.gated_forward(x, w_gate, w_up, w_down, activation, keep=True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, gate, up)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return *_ffi.gated_backward(dy, *ctx.saved_tensors, ctx.activation, ctx.needs_input_grad[:4]), None


def gated_feed_forward(x, w_gate, w_up, w_down, activation="silu"):
    """The block over the last dimension of ``x`` [..., D], differentiable (once, in reverse mode) in x and the weights: [..., O]."""
    if _ffi._dense.has_tangent(x, w_gate, w_up) or _ffi._dense.has_tangent(w_down, None, None):
        raise NotImplementedError("gated_feed_forward has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
        return _GatedFunction.apply(x, w_gate, w_up, w_down, activation)
    return _ffi.gated_forward(x, w_gate, w_up, w_down, activation)


class GatedFeedForward(torch.nn.Module):
    """The block as a module: matrices ``w_gate``, ``w_up`` [hidden, features] and ``w_down`` [out, hidden] (bf16, no biases), drawn uniformly as ``torch.nn.Linear`` draws its weight."""

    def __init__(self, features, hidden, out=None, activation="silu", device=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
        self.features, self.hidden, self.out, self.activation = int(features), int(hidden), int(features if out is None else out), activation
        for name, shape in (("w_gate", (self.hidden, self.features)), ("w_up", (self.hidden, self.features)), ("w_down", (self.out, self.hidden))):
            w = torch.nn.Parameter(torch.empty(shape, device=device, dtype=torch.bfloat16))
            with torch.no_grad():
                w.uniform_(-shape[1] ** -0.5, shape[1] ** -0.5)
            setattr(self, name, w)

    def forward(self, x):
        return gated_feed_forward(x, self.w_gate, self.w_up, self.w_down, self.activation)

    def extra_repr(self):
        return f"{self.features}, {self.hidden}, out={self.out}, activation={self.activation}"

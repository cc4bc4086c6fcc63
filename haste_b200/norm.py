"""Layer norm for the features that the fixed-fan-in layer reads: operator, autograd function and module.

    layer_norm(x, weight, bias, eps)      under autograd
    LayerNorm(features)                   module with torch.nn.LayerNorm's parameter names and state dict
    layer_norm_forward, _backward         the two kernels, for steps without an autograd graph

x and the gradient may be bf16 or fp32, weight and bias bf16 or fp32 whatever x is; statistics and sums are fp32.
"""
import torch

from . import ffi as _ffi
from .ffi import layer_norm_backward, layer_norm_forward  # noqa: F401


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _ffi.layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        want_w = weight is not None and ctx.needs_input_grad[1]
        want_b = ctx.bias_dtype is not None and ctx.needs_input_grad[2]
        dx, dw, db = _ffi.layer_norm_backward(dy, x, weight, mean, rstd, want_w, want_b, ctx.bias_dtype if weight is None else None)
        return dx if ctx.needs_input_grad[0] else None, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension of ``x`` [..., D], differentiable (once, in reverse mode) in x, weight and bias."""
    if _ffi._dense.has_tangent(x, weight, bias):
        raise NotImplementedError("layer_norm has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFunction.apply(x, weight, bias, float(eps))
    return _ffi.layer_norm_forward(x, weight, bias, float(eps), stats=False)


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension.  Parameters ``weight`` and ``bias`` as in ``torch.nn.LayerNorm`` (its state dicts load);
    ``dtype`` is theirs alone: fp32 parameters over bf16 features are fine."""

    def __init__(self, features, eps=1e-5, bias=True, device=None, dtype=None):
        super().__init__()
        self.features, self.eps = int(features), float(eps)
        self.weight = torch.nn.Parameter(torch.ones(self.features, device=device, dtype=dtype))
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(self.features, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.features}, eps={self.eps}, bias={self.bias is not None}"

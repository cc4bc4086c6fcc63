"""Token embedding for an encoder in front of the sparse layer: operator, autograd function and module.

    embedding(ids, table, scale)              under autograd
    Embedding(rows, features)                 module with torch.nn.Embedding's parameter name and state dict
    embedding_forward, embedding_backward     the kernels, for steps without an autograd graph

Tables are bf16 or fp32.  The gradient is dense, what ``AdamW`` takes; every row of it is summed in fp32 in the order of its tokens.
"""
import torch

from . import ffi as _ffi
from .ffi import embedding_backward, embedding_forward  # noqa: F401


class _EmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.told = table.shape[0], scale, padding_idx, table.dtype
        return _ffi.embedding_forward(ids, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        rows, scale, padding_idx, dtype = ctx.told
        return None, _ffi.embedding_backward(dy, ids, rows, scale, padding_idx, dtype), None, None


def embedding(ids, table, scale=1.0, padding_idx=None):
    """``scale * table[ids]``, differentiable (once, in reverse mode) in the table.  Row ``padding_idx`` gets no gradient."""
    if _ffi._dense.has_tangent(table, None, None):
        raise NotImplementedError("embedding has no forward-mode derivative")
    if padding_idx is not None and not -table.shape[0] <= padding_idx < table.shape[0]:
        raise RuntimeError(f"padding_idx {padding_idx} is no row of a table of {table.shape[0]}")
    if torch.is_grad_enabled() and table.requires_grad:
        return _EmbeddingFunction.apply(ids, table, float(scale), padding_idx)
    return _ffi.embedding_forward(ids, table, float(scale))


class Embedding(torch.nn.Module):
    """``rows`` vectors of ``features``, times ``scale``.  Parameter ``weight`` as in ``torch.nn.Embedding`` (its state dicts load), drawn as there: N(0, 1), the padding's row
    zeros."""

    def __init__(self, rows, features, padding_idx=None, scale=1.0, device=None, dtype=None):
        super().__init__()
        self.rows, self.features, self.scale = int(rows), int(features), float(scale)
        if padding_idx is not None and not -self.rows <= padding_idx < self.rows:
            raise ValueError(f"padding_idx {padding_idx} is no row of {self.rows}")
        self.padding_idx = padding_idx
        self.weight = torch.nn.Parameter(torch.empty(self.rows, self.features, device=device, dtype=dtype))
        with torch.no_grad():
            self.weight.normal_()
            if padding_idx is not None:
                self.weight[padding_idx].zero_()

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        return f"{self.rows}, {self.features}, padding_idx={self.padding_idx}, scale={self.scale}"

"""A training step of the output layer together with the dense part in front of it: projection, layer norm, sparse layer.

The reference puts a Linear between the encoder and the sparse layer (src/model.py:157-161, 242-243), trains it with the encoder's
optimizer and the sparse layer with its own (src/runner.py:129-137, 197).  ``ProjectedFusedStep`` is that with a layer norm behind the Linear,
which it needs, and without an autograd graph:

    a = h W^T + b         library GEMM
    x = layer norm of a   ``layer_norm_forward``
    fused sparse step     ``FusedFFIShard.step``: loss, the gradient of x, the sparse layer's update
    da                    ``layer_norm_backward``, with the gradients of the norm's weight and bias
    dW, db, dh            library GEMMs
    AdamW                 over W, b and the norm's parameters (and whatever else the optimizer holds), clipped by their joint norm; or Muon over W and AdamW over the rest
"""
import torch

from .norm import layer_norm_backward, layer_norm_forward


class ProjectedFusedStep:
    """``projection``: torch.nn.Linear [H -> P]; ``norm``: ``haste_b200.norm.LayerNorm(P)``; ``shard``: ``FusedFFIShard`` over P features;
    ``optimizer``: ``haste_b200.optim.AdamW`` that holds the parameters of the first two, or a list of optimizers that do (``Muon`` for the matrices beside it).  The
    projection and the features are bf16."""

    def __init__(self, projection, norm, shard, optimizer):
        if projection.out_features != norm.features or norm.features != shard.D:
            raise ValueError(f"the projection has {projection.out_features} outputs, the norm {norm.features} features, the sparse layer {shard.D}")
        if projection.weight.dtype != torch.bfloat16:
            raise ValueError("the projection must be bf16, as the sparse layer's features are")
        self.optimizer = optimizer
        held = {id(p) for o in self.optimizers for group in o.param_groups for p in group["params"]}
        if any(id(p) not in held for m in (projection, norm) for p in m.parameters()):
            raise ValueError("the optimizer must hold the projection's and the norm's parameters")
        self.projection, self.norm, self.shard = projection, norm, shard

    @property
    def optimizers(self):
        """``optimizer`` as a list: what ``update`` steps."""
        return list(self.optimizer) if isinstance(self.optimizer, (list, tuple)) else [self.optimizer]

    @torch.no_grad()
    def step(self, h, targets, want_loss=True):
        """``h`` bf16 [B, H], ``targets`` int32 [nnz, 2] (row, label).  Returns (dh bf16 [B, H], loss fp32 [1] or None); all parameters are updated
        in place.  The gradients stay in ``.grad``.  Other parameters of the optimizer take part in the step and its norm if they have a
        gradient: an encoder behind ``h`` that is trained by the same optimizer wants its backward pass between ``backward`` and ``update``."""
        dh, loss = self.backward(h, targets, want_loss)
        self.update()
        return dh, loss

    @torch.no_grad()
    def backward(self, h, targets, want_loss=True):
        """``step`` without the optimizer: the sparse layer is updated, the dense parameters have their gradients."""
        lin, norm = self.projection, self.norm
        a = torch.nn.functional.linear(h, lin.weight, lin.bias)
        x, mean, rstd = layer_norm_forward(a, norm.weight, norm.bias, norm.eps)
        dxt, loss = self.shard.step(x, targets, want_loss)
        # dxt is the fp32 gradient [P, B]
        da, dw, db = layer_norm_backward(dxt.t(), a, norm.weight, mean, rstd, want_bias=norm.bias is not None)
        norm.weight.grad = dw
        if norm.bias is not None:
            norm.bias.grad = db
        lin.weight.grad = da.t() @ h
        if lin.bias is not None:
            lin.bias.grad = da.sum(0, dtype=torch.float32).to(lin.bias.dtype)
        return da @ lin.weight, loss

    def update(self):
        for o in self.optimizers:
            o.step()

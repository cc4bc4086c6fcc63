"""AdamW over many tensors at once, for the dense parameters next to the sparse layer (``SRSgd`` trains the layer itself).

    AdamW(params, ...)          torch optimizer: bf16 (stochastic rounding, no fp32 copies) or fp32 parameters, moments in 32 or 8 bits,
                                gradients clipped by their global norm without a word from the host
    adamw_step, grad_norm       the kernels, on lists of tensors and flat moments
    quantize, dequantize        the 8-bit form of moments

The moments of a list of tensors lie in one buffer each, every tensor's at a multiple of 256 elements (``moment_offsets``).  In 8 bits
each 256 elements share an fp32 scale; codes are rounded stochastically, so that a second moment, which moves by a thousandth a
step, follows its gradients (include/haste_ffi.h has the format).
"""
import itertools
import operator
from typing import NamedTuple

import torch
from torch.optim import Optimizer

from . import _lib
from . import ffi as _ffi
from .ffi import MOMENT_BLOCK, _dense, grad_norm  # noqa: F401


class Quantized(NamedTuple):
    """A moment in 8 bits: codes uint8 [n], scales fp32 [n / 256]; ``signed``: a first moment, else a second."""
    codes: torch.Tensor
    scales: torch.Tensor
    signed: bool


def quantize(x, signed):
    """fp32 values (a multiple of 256) as ``Quantized``, to the nearest code."""
    return Quantized(*_ffi.quantize_moment(x, signed), signed)


def dequantize(moment, dtype=torch.float32):
    """The values a ``Quantized`` moment stands for."""
    return _ffi.dequantize_moment(moment.codes, moment.scales, moment.signed, dtype)


def moment_offsets(sizes):
    """Where the tensors of ``sizes`` elements start in a moment's buffer, and the buffer's size behind them."""
    at, out = 0, []
    for n in sizes:
        out.append(at)
        at += (n + MOMENT_BLOCK - 1) // MOMENT_BLOCK * MOMENT_BLOCK
    return out + [at]


def adamw_step(params, grads, exp_avg, exp_avg_sq, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, grad_scale=1.0, max_norm=None, norm=None,
               stochastic_rounding=True, seed=123, stream_index=0):
    """One AdamW step (decoupled weight decay) over lists of parameters, all bf16 or all fp32, and gradients (None: skipped), in place.

    ``exp_avg`` and ``exp_avg_sq`` are the flat moments: fp32 tensors, or ``Quantized``.  ``step`` counts from 1.  Gradients are
    multiplied with ``grad_scale``; with ``max_norm`` they are also clipped to that norm, which is returned (fp32 on the device; taken
    from ``norm`` where that is given, as when one norm is over the tensors of several calls), and a norm that is not finite leaves
    everything as it was.  Autograd takes what is written for changed in place.  Random bits follow from (seed, step, place in the moments, stream_index)."""
    quantized = isinstance(exp_avg, Quantized)
    if quantized != isinstance(exp_avg_sq, Quantized) or (quantized and not (exp_avg.signed and not exp_avg_sq.signed)):
        raise RuntimeError("both moments in 32 bits, or a signed and an unsigned Quantized")
    m, ms, v, vs = (*exp_avg[:2], *exp_avg_sq[:2]) if quantized else (exp_avg, None, exp_avg_sq, None)
    return _dense.adamw_step(params, grads, m, ms, v, vs, 8 if quantized else 32, step, lr, betas[0], betas[1], eps, weight_decay, grad_scale, norm, max_norm, seed,
                             stream_index, _lib.F_SR if stochastic_rounding else 0)


def _same(a, b):
    """Whether two lists hold the same objects."""
    return len(a) == len(b) and all(map(operator.is_, a, b))


class _Moments:
    """The flat moments of the parameters of one type in a parameter group, and each parameter's part of them."""

    def __init__(self, params, bits):
        self.params, self.bits = list(params), bits
        dev = self.params[0].device
        self.sizes = [p.numel() for p in self.params]
        self.offsets = moment_offsets(self.sizes)
        n = self.offsets[-1]
        if bits == 32:
            self.avg, self.sq = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
        else:
            zeros = lambda signed: Quantized(torch.zeros(n, dtype=torch.uint8, device=dev), torch.zeros(n // MOMENT_BLOCK, device=dev), signed)
            self.avg, self.sq = zeros(True), zeros(False)

    def views(self, i):
        """State entries of parameter i: views of the buffers."""
        p, a, b = self.params[i], self.offsets[i], self.offsets[i + 1]
        n = p.numel()
        if self.bits == 32:
            return {"exp_avg": self.avg[a:a + n].view(p.shape), "exp_avg_sq": self.sq[a:a + n].view(p.shape)}
        blocks = slice(a // MOMENT_BLOCK, b // MOMENT_BLOCK)
        return {"exp_avg": self.avg.codes[a:a + n].view(p.shape), "exp_avg_scale": self.avg.scales[blocks],
                "exp_avg_sq": self.sq.codes[a:a + n].view(p.shape), "exp_avg_sq_scale": self.sq.scales[blocks]}

    def adopt(self, i, old):
        """Take over saved entries of parameter i, in 8 or 32 bits, for what this has."""
        new = self.views(i)
        n, room = self.params[i].numel(), self.offsets[i + 1] - self.offsets[i]
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            x, s = old[name].to(new[name].device), old.get(name + "_scale")
            if tuple(x.shape) != tuple(new[name].shape):
                raise RuntimeError(f"saved {name} of shape {tuple(x.shape)} for a parameter of shape {tuple(new[name].shape)}")
            if (s is None) == (self.bits == 32):                       # the same form
                new[name].copy_(x)
                if s is not None:
                    new[name + "_scale"].copy_(s)
                continue
            flat = torch.zeros(room, dtype=torch.float32 if s is None else torch.uint8, device=x.device)
            flat[:n] = x.reshape(-1)
            if s is None:
                codes, scales = _ffi.quantize_moment(flat, signed)
                new[name].copy_(codes[:n].view(x.shape))
                new[name + "_scale"].copy_(scales)
            else:
                new[name].copy_(_ffi.dequantize_moment(flat, s.to(x.device).contiguous(), signed)[:n].view(x.shape))


class _Held:
    """A parameter's saved entries on their way through ``Optimizer.load_state_dict``, which casts the tensors that it finds."""

    def __init__(self, entries):
        self.entries = entries


def _hold(optimizer, state_dict):
    if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
        raise RuntimeError("state dicts with amsgrad or maximize are not supported")
    return dict(state_dict, state={k: _Held(v) for k, v in state_dict["state"].items()})


class AdamW(Optimizer):
    """AdamW with decoupled weight decay: one launch for all parameters of a group and type.

    bf16 parameters are rounded stochastically (``stochastic_rounding=False``: to nearest).  ``state_bits``: 32, or 8 for moments of one
    byte and a scale per 256 elements.  ``max_grad_norm``: gradients of all groups are clipped to this norm together; the last step's norm
    is in ``grad_norm`` (a scalar on the device), and a step whose norm is inf or NaN changes nothing but the step count.

    State dicts hold ``exp_avg`` and ``exp_avg_sq`` per parameter.  Those of ``torch.optim.AdamW`` load (not the other way round: that class
    counts its steps per parameter), and so do those of the other ``state_bits``.  Steps are counted per group: a parameter without a gradient is left alone, the count goes on."""

    _GROUP_KEYS = dict(state_bits=32, stochastic_rounding=True, seed=123, step_count=0)

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_grad_norm=None, stochastic_rounding=True, seed=123):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError("max_grad_norm must be positive")
        if not (lr >= 0 and weight_decay >= 0 and eps > 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError("lr and weight_decay must not be negative, eps must be positive, betas in [0, 1)")
        self.max_grad_norm, self.grad_norm = max_grad_norm, None
        self._moments, self._seen = {}, None                               # flat moments by group and type; the state's entries beside them
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, stochastic_rounding=stochastic_rounding,
                                      seed=seed, step_count=0))

    def __getstate__(self):
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm)

    def __setstate__(self, state):
        """From a pickle, a copy or ``load_state_dict``: the flat moments are made anew from the state's entries at the next step.  Loading, options
        that the saved groups lack are those of the groups that are replaced, and how moments are held is in any case."""
        replaced = self.__dict__.get("param_groups", ())
        super().__setstate__(state)
        self._moments, self._seen = {}, None
        self.__dict__.setdefault("max_grad_norm", None)
        self.__dict__.setdefault("grad_norm", None)
        for i, group in enumerate(self.param_groups):
            told = replaced[i] if i < len(replaced) else self._GROUP_KEYS
            if replaced:
                group["state_bits"] = told["state_bits"]
            held = {p: self.state[p].entries for p in group["params"] if isinstance(self.state.get(p), _Held)}
            for p, old in held.items():
                self.state[p] = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in old.items() if k.startswith("exp_avg")}
            if "step_count" not in group:
                group["step_count"] = max((int(old["step"]) for old in held.values() if "step" in old), default=0)
            for k in self._GROUP_KEYS:
                group.setdefault(k, told[k])
        for k, v in self.state.items():                                # entries of no parameter, which torch passes on
            if isinstance(v, _Held):
                self.state[k] = v.entries

    def load_state_dict(self, state_dict):
        """As ``Optimizer.load_state_dict``, but the moments keep their types (that one casts them to the parameters'), a state dict of
        ``torch.optim.AdamW`` brings its step count along, and ``state_bits`` stays what the constructor was told: the moments are converted."""
        last = self.register_load_state_dict_pre_hook(_hold)          # behind those of the user, which may replace the dict
        try:
            super().load_state_dict(state_dict)
        finally:
            last.remove()

    def _flat(self, index, group, dtype, params):
        """The moments of the group's parameters of one type; built at the first step, and again when they, their sizes or entries of the state
        were replaced."""
        m = self._moments.get((index, dtype))
        if m is not None and m.bits == group["state_bits"] and _same(m.params, params) and m.sizes == [p.numel() for p in params]:
            return m
        ours = {*map(id, params)}                                          # other buffers of theirs (of another type or group) hold them no longer
        self._moments = {k: other for k, other in self._moments.items() if ours.isdisjoint(map(id, other.params))}
        m = _Moments(params, group["state_bits"])
        for i, p in enumerate(params):
            state, views = self.state[p], m.views(i)
            if state:
                m.adopt(i, state)
            state.update(views)
            for gone in {"exp_avg_scale", "exp_avg_sq_scale"} & (state.keys() - views.keys()):
                del state[gone]
        self._moments[(index, dtype)], self._seen = m, None
        return m

    def _entries(self):
        """What the state holds: keys, entries, and what is in these."""
        entries = [s for s in self.state.values() if isinstance(s, dict)]
        return [*self.state, *entries, *itertools.chain.from_iterable(map(dict.values, entries))]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        all_grads = [[p.grad for p in group["params"]] for group in self.param_groups]
        norm = None
        if self.max_grad_norm is not None:
            grads = [g if g.is_contiguous() else g.contiguous() for grads in all_grads for g in grads if g is not None]
            if grads:
                norm = self.grad_norm = grad_norm(grads)
        if self._seen is None or not _same(self._seen, self._entries()):
            self._moments = {}                                             # something was taken away or replaced
        for index, (group, grads) in enumerate(zip(self.param_groups, all_grads)):
            group["step_count"] += 1
            params = group["params"]
            dtypes = [p.dtype for p in params]
            types = {t for t, g in zip(dtypes, grads) if g is not None}
            for k, dtype in enumerate((torch.bfloat16, torch.float32)):
                if dtype in types:
                    of = (lambda x: x) if dtypes.count(dtype) == len(dtypes) else lambda x: [a for a, t in zip(x, dtypes) if t == dtype]
                    self._step_type(group, self._flat(index, group, dtype, of(params)), of(grads), 2 * index + k, norm)
            if types - {torch.bfloat16, torch.float32}:
                raise RuntimeError(f"parameters must be torch.bfloat16 or torch.float32, got {types - {torch.bfloat16, torch.float32}}")
        if self._seen is None:
            self._seen = self._entries()
        return loss

    def _step_type(self, group, m, grads, stream_index, norm):
        params = [p if p.is_contiguous() else p.contiguous() for p in m.params]
        g_types = {g.dtype for g in grads if g is not None}
        for g_type in g_types:                                         # one launch, unless some gradients have another type
            part = grads if len(g_types) == 1 else [g if g is not None and g.dtype == g_type else None for g in grads]
            part = [g if g is None or g.is_contiguous() else g.contiguous() for g in part]
            adamw_step(params, part, m.avg, m.sq, step=group["step_count"], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], max_norm=self.max_grad_norm if norm is not None else None, norm=norm,
                       stochastic_rounding=group["stochastic_rounding"], seed=group["seed"], stream_index=stream_index)
        for p, q in zip(m.params, params):
            if p is not q:
                p.copy_(q)

"""AdamW over a list of tensors, for parameters that are not in an arena, with moments in 32 or 8 bits.

    adamw_step_   one step over lists of parameters, gradients and moments
    AdamW         an optimizer that keeps the moments (and fp32 masters of bf16 parameters)

The formulas and the 8-bit format stand beside the kernel's declaration (``include/bamboo_b200.h``, bb_adamw_list), the kernel in
``csrc/adamw.cu``.  An arena's flat buffers have ``lib.adam_step`` and ``post_training.adam_step_clipped``.
"""
import itertools
import operator

import torch

from . import lib as L
from .post_training import _gradient_of, _on_current

BLOCK = 256          # values of a tensor that share a scale where moments have 8 bits

_dtype_of = operator.attrgetter("dtype")
_sizes = torch.Tensor.numel
_address = torch.Tensor.data_ptr
_device_of = torch.Tensor.get_device
_contiguous = torch.Tensor.is_contiguous


def _column(tensors, name, count, dtypes, sizes, device):
    """A list that goes with the parameters: as many tensors, of one of these types, on the device, contiguous, of the same sizes."""
    if len(tensors) != count:
        raise ValueError(f"{name}: {len(tensors)} tensors for {count} parameters")
    if set(map(_device_of, tensors)) != {device}:
        raise L.BambooNativeError(f"{name}: expected on cuda:{device}, as the parameters")
    if not set(map(_dtype_of, tensors)) <= dtypes:
        raise L.BambooNativeError(f"{name}: {' or '.join(sorted(str(d) for d in dtypes))} expected")
    if not all(map(_contiguous, tensors)):
        raise L.BambooNativeError(f"{name}: contiguous tensors are expected")
    if sizes is not None and list(map(_sizes, tensors)) != sizes:
        raise ValueError(f"{name}: tensors of the parameters' sizes are expected")
    return map(_address, tensors)


_BF16, _FP32, _EITHER, _CODES = {torch.bfloat16}, {torch.float32}, {torch.bfloat16, torch.float32}, {torch.float8_e4m3fn}


def adamw_step_(params, grads, exp_avgs, exp_avg_sqs, *, scales=None, masters=None, step, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
                weight_decay=0.0, grad_scale=1.0, max_norm=0.0, sumsq=None, zero_grad=False, rounding="nearest"):
    """One AdamW step, number ``step`` (from 1), in place over lists of contiguous tensors; a parameter whose gradient is None is left out.

    ``params``: fp32, or bf16 with fp32 ``masters``.  ``grads``: bf16 or fp32.  Moments: fp32; or float8_e4m3fn with ``scales``, a fp32 tensor
    [2, blocks of 256 values] for each parameter, where ``exp_avg_sqs`` holds the SQUARE ROOT of the second moment.
    ``rounding`` of those codes: "nearest", or "stochastic", up or down by a hash of the step number and the value's place (the same call gives the same
    codes).  Training wants the latter: a step changes a root by (1 - beta2) / 2 of itself, and the nearest of codes that are 6 to 12 % apart stays the same,
    so that from beta2 = 0.99 on roots stop following their gradients (bb_adamw_list has figures).
    ``grad_scale`` multiplies the gradients first.  ``max_norm`` > 0: on gradients clipped to that norm over the whole list, or over ``sumsq``
    (sum of squares of unscaled gradients, fp64 [1], device) where it covers more; returns the norm before clipping (fp32 scalar, device).
    A captured call repeats its step number at every replay."""
    given = params = list(params)
    grads = list(grads)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if rounding not in ("nearest", "stochastic"):
        raise ValueError(f"rounding {rounding!r}: 'nearest' or 'stochastic'")
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError(f"beta1 {beta1}, beta2 {beta2}: from 0 to below 1")
    lists = [grads, *(None if column is None else list(column) for column in (exp_avgs, exp_avg_sqs, scales, masters))]
    for name, column in zip(("grads", "exp_avgs", "exp_avg_sqs", "scales", "masters"), lists):
        if column is not None and len(column) != len(params):
            raise ValueError(f"{name}: {len(column)} tensors for {len(params)} parameters")
    sizes = list(map(_sizes, params))
    seeds = range(1, len(params) + 1)
    if not all(sizes) or type(None) in set(map(type, grads)):
        keep = [i for i, g in enumerate(grads) if g is not None and sizes[i]]
        params, sizes, seeds = [params[i] for i in keep], [sizes[i] for i in keep], [i + 1 for i in keep]
        lists = [None if column is None else [column[i] for i in keep] for column in lists]
    grads, exp_avgs, exp_avg_sqs, scales, masters = lists
    count = len(params)
    if not count:
        if not max_norm > 0:
            return None
        if sumsq is None:           # (on the device, as of any other list)
            return torch.zeros((), device=given[0].device if given else "cuda" if torch.cuda.is_available() else "cpu")
        return (sumsq.detach().sqrt() * grad_scale).to(torch.float32).reshape(())
    _on_current(params[0], "params")
    device = params[0].get_device()
    moments = _FP32 if scales is None else _CODES
    addresses = _column(params, "params", count, _FP32 if masters is None else _BF16, None, device)
    if scales is not None and list(map(_sizes, scales)) != [2 * -(-n // BLOCK) for n in sizes]:
        raise ValueError("scales: [2, blocks of 256 values] for every parameter")
    if sumsq is not None and (sumsq.get_device() != device or sumsq.dtype != torch.float64):
        raise L.BambooNativeError("sumsq is fp64, on the parameters' device")
    nothing = itertools.repeat(0)
    first = _column(exp_avgs, "exp_avgs", count, moments, sizes, device)
    second = _column(exp_avg_sqs, "exp_avg_sqs", count, moments, sizes, device)
    full = nothing if masters is None else _column(masters, "masters", count, _FP32, sizes, device)
    scaled = nothing if scales is None else _column(scales, "scales", count, _FP32, None, device)
    fields = itertools.chain.from_iterable(zip(
        addresses, full, _column(grads, "grads", count, _EITHER, sizes, device), first, second, scaled, sizes,
        map(L.dtype_codes().get, map(_dtype_of, grads)), seeds if rounding == "stochastic" else nothing))
    table = L.adamw_tensors(fields, count)
    if L.adamw_overlaps(table, count, zero_grad):
        raise ValueError("a tensor stands twice among params, moments, scales and masters (and gradients that are zeroed), or shares memory with another")
    norm = scratch = None
    if max_norm > 0:            # (no buffer that calls share: a captured one keeps its own)
        norm = torch.empty((), dtype=torch.float32, device=params[0].device)
        scratch = torch.empty(L.grad_norm_bytes(), dtype=torch.uint8, device=params[0].device)
    L.adamw_list(table, count, lr=float(lr), beta1=float(beta1), beta2=float(beta2), eps=float(eps), step=int(step),
                 weight_decay=float(weight_decay), grad_scale=float(grad_scale), zero_grad=zero_grad, max_norm=float(max_norm), sumsq=sumsq, norm=norm,
                 scratch=scratch)
    torch.autograd.graph.increment_version(params + grads if zero_grad else params)
    return norm


class AdamW:
    """``adamw_step_`` over ``params`` (leaf tensors, fp32 or all bf16), with the state that it needs.

    ``state_bits``: 32, or 8 for moments of one byte each, their codes rounded "stochastic".  bf16 parameters get fp32 masters, which the steps are taken on.  ``max_norm`` > 0 clips
    the gradients' global norm.  ``step()`` reads ``main_grad`` of a parameter where it has one, else ``grad``."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, *, state_bits=32, max_norm=0.0):
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: 8 or 32")
        dtypes = {p.dtype for p in self.params}
        if len(dtypes) != 1 or not dtypes <= _EITHER:
            raise L.BambooNativeError(f"parameters are all fp32 or all bf16, got {sorted(map(str, dtypes))}")
        self.lr, self.betas, self.eps, self.weight_decay, self.max_norm, self.state_bits = lr, tuple(betas), eps, weight_decay, max_norm, state_bits
        self.step_count = 0
        moment = torch.float8_e4m3fn if state_bits == 8 else torch.float32
        data = [p.detach() for p in self.params]
        self.masters = [p.float() for p in data] if dtypes == _BF16 else None
        self.exp_avgs = [torch.zeros(p.shape, dtype=moment, device=p.device) for p in data]
        self.exp_avg_sqs = [torch.zeros(p.shape, dtype=moment, device=p.device) for p in data]
        self.scales = [torch.zeros(2, -(-p.numel() // BLOCK), device=p.device) for p in data] if state_bits == 8 else None

    def step(self, *, grad_scale=1.0, sumsq=None):
        """One step; returns the norm before clipping (fp32 scalar, device) where the optimizer clips, else None."""
        if torch.cuda.is_current_stream_capturing():
            raise L.BambooNativeError("AdamW.step counts its steps on the host and cannot be captured; adamw_step_ can, with one step number")
        with torch.no_grad():
            data = [p.detach() for p in self.params]
            norm = adamw_step_(data, [_gradient_of(p) if p.requires_grad else None for p in self.params], self.exp_avgs, self.exp_avg_sqs,
                               scales=self.scales, masters=self.masters, step=self.step_count + 1, rounding="stochastic", lr=self.lr, beta1=self.betas[0],
                               beta2=self.betas[1], eps=self.eps, weight_decay=self.weight_decay, grad_scale=grad_scale, max_norm=self.max_norm, sumsq=sumsq)
        self.step_count += 1
        return norm

    def zero_grad(self):
        for p in self.params:
            main = getattr(p, "main_grad", None)
            if main is not None:
                main.zero_()
            p.grad = None

    def state_dict(self):
        """Everything a step depends on but the parameters (the masters of bf16 ones included); tensors are the optimizer's own."""
        return {"step": self.step_count, "state_bits": self.state_bits, "lr": self.lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay,
                "max_norm": self.max_norm, "exp_avgs": self.exp_avgs, "exp_avg_sqs": self.exp_avg_sqs, "scales": self.scales, "masters": self.masters}

    def load_state_dict(self, state):
        if state["state_bits"] != self.state_bits:
            raise ValueError(f"moments of {state['state_bits']} bits for an optimizer of {self.state_bits}")
        for name in ("exp_avgs", "exp_avg_sqs", "scales", "masters"):
            own, given = getattr(self, name), state[name]
            if (own is None) != (given is None) or (own is not None and [t.shape for t in own] != [t.shape for t in given]):
                raise ValueError(f"{name}: not those of these parameters")
        for name in ("exp_avgs", "exp_avg_sqs", "scales", "masters"):
            for to, t in zip(getattr(self, name) or (), state[name] or ()):
                to.copy_(t)
        self.step_count = int(state["step"])
        self.lr, self.betas, self.eps = state["lr"], tuple(state["betas"]), state["eps"]
        self.weight_decay, self.max_norm = state["weight_decay"], state["max_norm"]

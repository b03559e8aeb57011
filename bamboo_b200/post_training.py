"""Post-training of the vocabulary models: what follows token cross entropy when a model learns from preferences or rewards.

    token_logprobs      log-probabilities of given tokens, from logits
    head_logprobs       the same from hidden states and the vocabulary projection, whose logits are never stored
    preference_loss     paired preference loss over token log-probabilities (reference against policy)
    policy_loss         clipped policy loss with a KL term over token log-probabilities
    PreferenceLoss,     the two from logits, as ``loss_fn`` of a ``PipelineModule`` (labels are a tuple of tensors) or in one
    PolicyLoss          call without autograd (``loss_and_grad``)
    clip_grad_norm_,    global norm over a list of gradients, clipping in place, and the Adam step that clips;
    global_grad_norm,   ``gradient_clipping`` in the engine's configuration uses the same kernels
    adam_step_clipped

Formulas stand beside the kernels' declarations (``include/bamboo_b200.h``) and in ``csrc/post_training.cu``.  Tokens whose target is
``ignore_index`` (prompts, padding) count nowhere and get no gradient; what stands at their places in logits, log-probabilities and
advantages may be anything, NaN and infinities included.  Everything runs on the current stream, nothing synchronises, and there is no
fallback: CPU tensors are refused.  Gradients have no gradient of their own (it raises), and what is written over (``inplace``) is known to autograd.
"""
import functools
import itertools
import operator

import torch
from torch import nn

from . import lib as L


# ----------------------------------------------------------------------------------- arguments
def _on_current(t, name):
    """The kernels run on the current device's stream: tensors of another device are refused, as are CPU tensors."""
    where = t.get_device()
    if where < 0:
        raise L.BambooNativeError(f"{name}: expected a CUDA tensor; the sm_100a kernels have no CPU fallback")
    if where != torch._C._cuda_getDevice():
        raise L.BambooNativeError(f"{name}: on cuda:{where}, but cuda:{torch._C._cuda_getDevice()} is the current device")


def _rows(logits, vocab):
    """(logits, rows, vocab): contiguous logits [..., cols] as they are, others as [rows, cols] with unit inner stride (a copy only where
    their strides ask for one)."""
    _on_current(logits, "logits")
    cols = logits.shape[-1]
    if vocab is None:
        vocab = cols
    if not 0 < vocab <= cols:
        raise ValueError(f"vocab {vocab} does not fit logits with {cols} columns")
    if not logits.is_contiguous():
        logits = logits.detach().reshape(-1, cols)
        if logits.stride(1) != 1 or (logits.shape[0] > 1 and logits.stride(0) < cols):
            logits = logits.contiguous()
    return logits, logits.numel() // cols, vocab


def _flat(t, name, numel, dtype, device):
    """A per-token (or per-sequence) tensor as contiguous memory of the given type, whatever its shape."""
    if t.dtype is dtype and t.numel() == numel and t.device == device and t.is_contiguous():
        return t
    if t.device != device:
        raise L.BambooNativeError(f"{name}: on {t.device}, the logits are on {device}")
    if t.numel() != numel:
        raise ValueError(f"{name}: {t.numel()} values for {numel}")
    t = t.detach().reshape(-1)
    if t.dtype != dtype:
        if dtype == torch.int64 and t.is_floating_point():
            raise TypeError(f"{name}: token ids are integers, got {t.dtype}")
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _row_grad(grad, rows):
    """What autograd hands to a backward pass, as contiguous fp32."""
    return grad if grad.is_contiguous() and grad.dtype is torch.float32 else _flat(grad, "gradient", rows, torch.float32, grad.device)


def _geometry(targets, offsets):
    """(sequences, offsets as int64): the rows of 2-D targets, or what the offsets delimit in 1-D ones."""
    if offsets is not None:
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("offsets: one more than there are sequences, 1-D")
        return offsets.numel() - 1, _flat(offsets, "offsets", offsets.numel(), torch.int64, targets.device)
    if targets.dim() != 2:
        raise ValueError("targets [sequences, tokens], or 1-D with offsets")
    return targets.shape[0], None


def _inverse(temperature):
    if not temperature > 0:
        raise ValueError(f"temperature has to be positive, got {temperature}")
    return 1.0 / float(temperature)


def _overwritten(t):
    """Tell autograd that a kernel wrote over ``t``: what kept it for a backward pass raises instead of reading something else."""
    torch.autograd.graph.increment_version(t)


def _wants_grad(t):
    return t.requires_grad and torch.is_grad_enabled()


class _NoSecondDerivative(torch.autograd.Function):
    """A gradient as it is; an error where it is differentiated."""

    @staticmethod
    def forward(ctx, grad, anchor):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("the post-training functions are once_differentiable: their gradients have no gradient of their own")


def _once_differentiable(backward):
    """For a backward pass of kernels: under ``create_graph`` its gradients would count as constants.  (torch's decorator of that name lets them
    where the incoming gradient is one.)"""
    @functools.wraps(backward)
    def once(ctx, grad):
        if not torch.is_grad_enabled():
            return backward(ctx, grad)
        with torch.no_grad():
            grads = backward(ctx, grad)
        return tuple(g if g is None else _NoSecondDerivative.apply(g, torch.empty(0, requires_grad=True)) for g in grads)
    return once


# ----------------------------------------------------------------------------------- token log-probabilities
def _logprobs(lg, rows, tg, vocab, scale, ignore_index, shape=None, keep=True):
    """(log-probabilities, softmax sums for the backward pass unless ``keep`` is off)"""
    logp = torch.empty(rows if shape is None else shape, dtype=torch.float32, device=lg.device)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=lg.device) if keep else None
    if rows:
        L.token_logprob_fwd(lg, tg, logp, stats, vocab, scale, ignore_index)
    return logp, stats


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, vocab, scale, ignore_index, inplace):
        lg, rows, vocab = _rows(logits, vocab)
        tg = _flat(targets, "targets", rows, torch.int64, lg.device)
        logp, stats = _logprobs(lg, rows, tg, vocab, scale, ignore_index, targets.shape)
        ctx.args = rows, vocab, scale, ignore_index, inplace, stats, None if lg is logits else logits.shape
        ctx.save_for_backward(lg, tg)
        return logp

    @staticmethod
    @_once_differentiable
    def backward(ctx, grad):
        lg, tg = ctx.saved_tensors
        rows, vocab, scale, ignore_index, inplace, stats, shape = ctx.args
        out = lg.detach() if inplace else torch.empty_like(lg)
        if rows:
            L.token_logprob_bwd(lg, tg, stats, _row_grad(grad, rows), out, vocab, scale, ignore_index)
            if inplace:
                _overwritten(lg)
        return out if shape is None else out.view(shape), None, None, None, None, None


def token_logprobs(logits, targets, vocab=None, *, temperature=1.0, ignore_index=-100, inplace=False):
    """Log-probabilities (fp32, shaped like ``targets``) of ``targets`` under softmax(logits[..., :vocab] / temperature).

    ``logits`` [..., cols] bf16 or fp32; columns from ``vocab`` on are padding and get a zero gradient.  Ignored targets give 0.
    ``inplace``: the gradient overwrites the logits in the backward pass (once)."""
    scale = _inverse(temperature)
    if _wants_grad(logits):
        return _TokenLogprobsFn.apply(logits, targets, vocab, scale, ignore_index, inplace)
    lg, rows, vocab = _rows(logits, vocab)
    tg = _flat(targets, "targets", rows, torch.int64, lg.device)
    return _logprobs(lg, rows, tg, vocab, scale, ignore_index, targets.shape, keep=False)[0]


# ----------------------------------------------------------------------------------- through the vocabulary projection
# Bytes of logit gradient that exist at a time in the backward pass of head_logprobs
HEAD_GRAD_BYTES = 256 << 20


@functools.lru_cache(maxsize=256)
def _head_desc(rows, vocab, hidden, ld_hidden, ld_weight, scale, ignore_index):
    return L.HeadDesc(rows=rows, vocab=vocab, hidden=hidden, ld_hidden=ld_hidden, ld_weight=ld_weight, scale=scale, ignore_index=ignore_index)


def _aligned_rows(t, n):
    """``t`` as [rows, n] with 16-byte rows (a copy only where its layout asks for one)."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, n
    t = t.detach().reshape(-1, n)
    if t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < n or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(0)


def _head_operands(hidden, weight, targets, vocab, scale, ignore_index):
    for name, t in (("hidden", hidden), ("weight", weight)):
        _on_current(t, name)
        if t.dtype != torch.bfloat16:
            raise L.BambooNativeError(f"{name}: bf16 expected, got {t.dtype}")
    n = hidden.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != n:
        raise ValueError(f"weight {tuple(weight.shape)} for hidden states of {n}")
    if vocab is None:
        vocab = weight.shape[0]
    if not 0 < vocab <= weight.shape[0]:
        raise ValueError(f"vocab {vocab} does not fit a weight of {weight.shape[0]} rows")
    if n == 0 or n % 8:
        raise ValueError(f"hidden size {n}: a multiple of 8 is needed (16-byte rows)")
    (h, ld_h), (w, ld_w) = _aligned_rows(hidden, n), _aligned_rows(weight, n)
    rows = h.numel() // n
    return _head_desc(rows, vocab, n, ld_h, ld_w, scale, ignore_index), h, w, _flat(targets, "targets", rows, torch.int64, h.device)


def _head_forward(desc, h, w, tg, shape):
    logp = torch.empty(shape, dtype=torch.float32, device=h.device)
    stats = torch.empty(desc.rows, 2, dtype=torch.float32, device=h.device)
    if desc.rows:
        L.head_logprob_fwd(desc, h, w, tg, logp, stats)
    return logp, stats


class _HeadLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, vocab, scale, ignore_index):
        desc, h, w, tg = _head_operands(hidden, weight, targets, vocab, scale, ignore_index)
        logp, stats = _head_forward(desc, h, w, tg, targets.shape)
        ctx.args = desc, weight, hidden.shape, stats
        ctx.save_for_backward(h, w, tg)
        return logp

    @staticmethod
    @_once_differentiable
    def backward(ctx, grad):
        h, w, tg = ctx.saved_tensors
        desc, weight, shape, stats = ctx.args
        dev, rows, n, vocab = h.device, desc.rows, desc.hidden, desc.vocab
        need_h, need_w = ctx.needs_input_grad[:2]
        main = getattr(weight, "main_grad", None) if need_w else None
        dh = torch.empty(shape, dtype=torch.bfloat16, device=dev) if need_h else None
        dw = torch.empty(weight.shape, dtype=torch.bfloat16, device=dev) if need_w and main is None else None
        if dw is not None and (vocab < dw.shape[0] or not rows):
            dw[vocab if rows else 0:].zero_()
        if rows:
            # vocabulary entries in pieces, so that the gradient of the logits never exists whole; a multiple of 256, the widest tile
            piece = max(2048, HEAD_GRAD_BYTES // (2 * rows) // 256 * 256)
            width = (min(piece, vocab) + 63) // 64 * 64        # rows on lines of their own
            parts = L.head_bwd_parts(desc, piece) if need_h else 0
            scratch = torch.empty(L.head_bwd_scratch(desc, width, need_w, parts)[2], dtype=torch.uint8, device=dev)
            L.head_logprob_bwd(desc, h, w, tg, stats, _row_grad(grad, rows), dh, parts, dw, main, piece, width, scratch)
        return dh, dw, None, None, None, None


def head_logprobs(hidden, weight, targets, vocab=None, *, temperature=1.0, ignore_index=-100):
    """``token_logprobs(hidden @ weight.T, targets, vocab)`` without storing the logits: bf16 ``hidden`` [..., n] and ``weight`` [>= vocab, n],
    n a multiple of 8, fp32 logits inside.

    The backward pass computes the logits again, in pieces of the vocabulary.  The weight's gradient is added to ``weight.main_grad`` where
    the weight belongs to an arena, like the layers' gradients, and returned to autograd (bf16) otherwise."""
    scale = _inverse(temperature)
    if _wants_grad(hidden) or _wants_grad(weight):
        return _HeadLogprobsFn.apply(hidden, weight, targets, vocab, scale, ignore_index)
    return _head_forward(*_head_operands(hidden, weight, targets, vocab, scale, ignore_index), targets.shape)[0]


# ----------------------------------------------------------------------------------- losses over log-probabilities
# (descriptors are kept: making one costs the host as much as a launch.  They are known by plain numbers: a constant that is a tensor may hold
# another value at the next call)
@functools.lru_cache(maxsize=256)
def _kept_preference_desc(tokens, sequences, beta, form, label_smoothing, average, ignore_index):
    if form not in L.PREFERENCE_FORMS:
        raise ValueError(f"form {form!r}: one of {sorted(L.PREFERENCE_FORMS)}")
    if sequences % 2:
        raise ValueError(f"{sequences} sequences: preferences come in pairs (preferred, rejected)")
    return L.PreferenceDesc(tokens=tokens, sequences=sequences, form=L.PREFERENCE_FORMS[form], beta=beta, label_smoothing=label_smoothing,
                            average=average, ignore_index=ignore_index)


def _preference_desc(tokens, sequences, beta, form, label_smoothing, average, ignore_index):
    return _kept_preference_desc(tokens, sequences, float(beta), form, float(label_smoothing), int(average), int(ignore_index))


@functools.lru_cache(maxsize=256)
def _kept_policy_desc(tokens, sequences, advantages, clip_low, clip_high, kl_coef, reduction, ignore_index):
    if reduction not in L.POLICY_REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: one of {sorted(L.POLICY_REDUCTIONS)}")
    per_sequence = advantages == sequences and tokens != sequences
    return L.PolicyDesc(tokens=tokens, sequences=sequences, reduction=L.POLICY_REDUCTIONS[reduction], clip_low=clip_low, clip_high=clip_high,
                        kl_coef=kl_coef, advantage_per_sequence=int(per_sequence), ignore_index=ignore_index)


def _policy_desc(tokens, sequences, offsets, advantages, clip_low, clip_high, kl_coef, reduction, ignore_index):
    count = advantages.numel()
    if count != tokens and (count != sequences or offsets is not None):
        how = ("one per token or per sequence" if offsets is None else
               "one per token here (repeat_interleave those of the sequences); one per sequence goes with sequences of one length, as 2-D targets")
        raise ValueError(f"advantages: {count} values for {tokens} tokens in {sequences} sequences; {how}")
    return _kept_policy_desc(tokens, sequences, count, float(clip_low), float(clip_high), float(kl_coef), reduction, int(ignore_index))


class _ScaledFn(torch.autograd.Function):
    """A loss whose gradient was computed with it: backward multiplies by what arrives."""

    @staticmethod
    def forward(ctx, logps, loss, row_grad):
        ctx.save_for_backward(row_grad)
        return loss.clone()

    @staticmethod
    @_once_differentiable
    def backward(ctx, grad):
        (row_grad,) = ctx.saved_tensors
        return row_grad * grad, None, None


def preference_loss(logps, ref_logps, targets, *, beta=0.1, form="sigmoid", label_smoothing=0.0, average=False, offsets=None,
                    ignore_index=-100):
    """(loss, rewards [sequences]) over token log-probabilities, with autograd for ``logps``.

    Sequences 2i (preferred) and 2i + 1 (rejected) are a pair: the rows of 2-D ``targets``, or ``offsets`` [sequences + 1] into 1-D ones.
    ``ref_logps``: the reference model's, or None.  ``form``: "sigmoid" (with ``label_smoothing``), "hinge" or "squared"; ``average``:
    mean instead of sum over a sequence's tokens."""
    sequences, offsets = _geometry(targets, offsets)
    lp = _flat(logps, "logps", targets.numel(), torch.float32, targets.device)
    loss, rewards, row_grad = _preference(lp, ref_logps, targets, offsets, _preference_desc(
        lp.numel(), sequences, beta, form, label_smoothing, average, ignore_index))
    if _wants_grad(logps):
        loss = _ScaledFn.apply(logps, loss, row_grad.view(logps.shape))
    return loss, rewards


def _preference(lp, ref, targets, offsets, desc):
    _on_current(lp, "logps")
    n, dev = desc.tokens, lp.device
    tg = _flat(targets, "targets", n, torch.int64, dev)
    ref = None if ref is None else _flat(ref, "ref_logps", n, torch.float32, dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rewards = torch.empty(desc.sequences, dtype=torch.float32, device=dev)
    row_grad = torch.empty_like(lp)
    L.preference_loss(desc, lp, ref, tg, offsets, loss, rewards, row_grad)
    return loss, rewards, row_grad


def policy_loss(logps, old_logps, advantages, targets, *, ref_logps=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="token",
                offsets=None, ignore_index=-100):
    """(loss, stats) over token log-probabilities, with autograd for ``logps``; stats [2]: mean KL, share of clipped tokens.

    ``old_logps``: those of the policy that sampled the tokens (None: this very policy).  ``advantages``: per token, or per sequence of
    2-D ``targets``.  ``reduction``: "token" averages over all counted tokens, "sequence" averages the sequences' means."""
    sequences, offsets = _geometry(targets, offsets)
    lp = _flat(logps, "logps", targets.numel(), torch.float32, targets.device)
    _on_current(lp, "logps")
    desc = _policy_desc(lp.numel(), sequences, offsets, advantages, clip_low, clip_high, kl_coef, reduction, ignore_index)
    loss, stats = torch.empty((), dtype=torch.float32, device=lp.device), torch.empty(2, dtype=torch.float32, device=lp.device)
    row_grad = torch.empty_like(lp)
    L.policy_loss(desc, lp, *_policy_inputs(desc, old_logps, advantages, ref_logps, targets, lp.device), offsets, loss, stats, row_grad)
    if _wants_grad(logps):
        loss = _ScaledFn.apply(logps, loss, row_grad.view(logps.shape))
    return loss, stats


def _policy_inputs(desc, old, advantages, ref, targets, dev):
    n = desc.tokens
    return (None if old is None else _flat(old, "old_logps", n, torch.float32, dev),
            _flat(advantages, "advantages", desc.sequences if desc.advantage_per_sequence else n, torch.float32, dev),
            None if ref is None else _flat(ref, "ref_logps", n, torch.float32, dev),
            _flat(targets, "targets", n, torch.int64, dev))


# ----------------------------------------------------------------------------------- losses from logits
class _LogitsLossFn(torch.autograd.Function):
    """loss_fn(logits, labels) whose gradient the loss function makes itself (``_forward``, ``_backward``)."""

    @staticmethod
    def forward(ctx, logits, loss_fn, labels, offsets):
        ctx.loss_fn, ctx.shape = loss_fn, logits.shape
        return loss_fn._forward(ctx, logits, labels, offsets)

    @staticmethod
    @_once_differentiable
    def backward(ctx, grad):
        out = ctx.loss_fn._backward(ctx, grad.reshape(1).to(torch.float32).contiguous())
        return out.view(ctx.shape), None, None, None


class PreferenceLoss:
    """Paired preference loss from logits: ``loss_fn(logits, (targets, ref_logps))`` for the last stage; reference-free with targets alone.

    ``vocab``: real logit columns (the rest is padding; None: all).  The gradient overwrites the logits in the backward pass (one, then) unless
    ``inplace`` is off.  ``rewards`` keeps the last call's beta-scaled log-ratios per sequence (device)."""

    def __init__(self, vocab, *, beta=0.1, form="sigmoid", label_smoothing=0.0, average=False, temperature=1.0, ignore_index=-100,
                 inplace=True):
        self.vocab, self.scale, self.ignore_index, self.inplace = vocab, _inverse(temperature), ignore_index, inplace
        self.form = (beta, form, label_smoothing, average)
        self.rewards = None

    def _prepare(self, logits, labels, offsets):
        targets, ref = labels if isinstance(labels, (tuple, list)) else (labels, None)
        lg, rows, vocab = _rows(logits, self.vocab)
        sequences, offsets = _geometry(targets, offsets)
        tg = _flat(targets, "targets", rows, torch.int64, lg.device)
        ref = None if ref is None else _flat(ref, "ref_logps", rows, torch.float32, lg.device)
        return lg, vocab, tg, ref, offsets, _preference_desc(rows, sequences, *self.form, self.ignore_index)

    def _run(self, lg, vocab, tg, ref, offsets, desc, dlogits=None, grad_scale=1.0, stats=None, row_grad=None):
        loss = torch.empty((), dtype=torch.float32, device=lg.device)
        self.rewards = torch.empty(desc.sequences, dtype=torch.float32, device=lg.device)
        return L.preference_loss_logits(desc, lg, tg, vocab, ref, offsets, loss, self.rewards, dlogits, self.scale, grad_scale, stats, row_grad)

    def _forward(self, ctx, logits, labels, offsets):
        lg, vocab, tg, *rest = self._prepare(logits, labels, offsets)
        lg, n = lg.detach(), tg.numel()
        stats, row_grad = torch.empty(n, 2, dtype=torch.float32, device=lg.device), torch.empty(n, dtype=torch.float32, device=lg.device)
        loss = self._run(lg, vocab, tg, *rest, stats=stats, row_grad=row_grad)
        ctx.args = vocab, self.scale, self.ignore_index, self.inplace
        ctx.save_for_backward(lg, tg, stats, row_grad)
        return loss

    @staticmethod
    def _backward(ctx, grad):
        lg, tg, stats, row_grad = ctx.saved_tensors
        vocab, scale, ignore_index, inplace = ctx.args
        out = lg if inplace else torch.empty(lg.shape, dtype=lg.dtype, device=lg.device)
        L.token_logprob_bwd(lg, tg, stats, row_grad, out, vocab, scale, ignore_index, grad_scale_dev=grad)
        if inplace:
            _overwritten(lg)
        return out

    def __call__(self, logits, labels, offsets=None):
        if _wants_grad(logits):
            return _LogitsLossFn.apply(logits, self, labels, offsets)
        return self._run(*self._prepare(logits, labels, offsets))

    def loss_and_grad(self, logits, labels, *, offsets=None, out=None, grad_scale=1.0):
        """(loss, rewards, gradient of the logits times ``grad_scale``) without autograd; ``out`` receives the gradient (the logits
        themselves are allowed)."""
        args = self._prepare(logits, labels, offsets)
        d, grad = _gradient_buffer(logits, out)
        return self._run(*args, d, grad_scale), self.rewards, grad


def _gradient_buffer(logits, out):
    """(tensor for the kernels, tensor for the caller) of the gradient."""
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return out, out
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out: a tensor like the logits is expected")
    d = out.detach() if out.is_contiguous() else out.detach().view(-1, out.shape[-1])
    if d.stride(-1) != 1:
        raise ValueError("out: rows with unit stride are expected")
    return d, out


def _policy_both(lg, vocab, desc, inputs, offsets, d, scale, grad_scale):
    """(loss, stats) from logits, and their gradient into ``d``."""
    old, advantages, ref, tg = inputs
    loss = torch.empty((), dtype=torch.float32, device=lg.device)
    stats = torch.empty(2, dtype=torch.float32, device=lg.device)
    L.policy_loss_logits(desc, lg, tg, vocab, old, advantages, ref, offsets, loss, stats, None, d, scale, grad_scale)
    return loss, stats


class PolicyLoss:
    """Clipped policy loss from logits: ``loss_fn(logits, (targets, old_logps, advantages[, ref_logps]))`` for the last stage.

    The gradient of a row of logits needs that row alone, so loss and gradient come from one pass in the forward call, for an upstream
    gradient of ``grad_scale`` (the pipeline engine sets it to 1 / micro-batches); a different upstream gradient costs a pass
    over the gradient in the backward call.  It overwrites the logits IN THE FORWARD call unless ``inplace`` is off; a second backward
    pass over a kept graph is then an error, and makes the gradient again where it is off.  ``stats`` keeps the last call's mean KL and
    share of clipped tokens (device)."""

    def __init__(self, vocab, *, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="token", temperature=1.0, ignore_index=-100,
                 inplace=True):
        self.vocab, self.scale, self.ignore_index, self.inplace = vocab, _inverse(temperature), ignore_index, inplace
        self.form = (clip_low, clip_high, kl_coef, reduction)
        self.grad_scale = 1.0
        self.stats = None

    def _prepare(self, logits, labels, offsets):
        targets, old, advantages = labels[:3]
        ref = labels[3] if len(labels) > 3 else None
        lg, rows, vocab = _rows(logits, self.vocab)
        sequences, offsets = _geometry(targets, offsets)
        desc = _policy_desc(rows, sequences, offsets, advantages, *self.form, self.ignore_index)
        return lg, vocab, desc, _policy_inputs(desc, old, advantages, ref, targets, lg.device), offsets

    def _both(self, lg, vocab, desc, inputs, offsets, d, grad_scale):
        loss, self.stats = _policy_both(lg, vocab, desc, inputs, offsets, d, self.scale, grad_scale)
        return loss

    def _forward(self, ctx, logits, labels, offsets):
        lg, vocab, desc, inputs, offsets = self._prepare(logits, labels, offsets)
        lg = lg.detach()
        ctx.args = vocab, desc, self.scale, self.grad_scale, self.inplace
        d = lg if self.inplace else torch.empty(lg.shape, dtype=lg.dtype, device=lg.device)
        loss = self._both(lg, vocab, desc, inputs, offsets, d, self.grad_scale)
        if self.inplace:
            _overwritten(lg)
            ctx.save_for_backward(d)
        else:
            # (the first backward pass hands its gradient out; what further ones over a kept graph need to make theirs)
            ctx.made = d
            ctx.save_for_backward(lg, offsets, *inputs)
        return loss

    @staticmethod
    def _backward(ctx, grad):
        vocab, desc, scale, made_for, inplace = ctx.args
        if inplace:
            (d,) = ctx.saved_tensors
        else:
            d, ctx.made = ctx.made, None
            if d is None:
                lg, offsets, *inputs = ctx.saved_tensors
                d = torch.empty(lg.shape, dtype=lg.dtype, device=lg.device)
                _policy_both(lg, vocab, desc, inputs, offsets, d, scale, made_for)
        L.rescale(d, grad, made_for)
        if inplace:
            _overwritten(d)
        return d

    def __call__(self, logits, labels, offsets=None):
        if _wants_grad(logits):
            return _LogitsLossFn.apply(logits, self, labels, offsets)
        lg, vocab, desc, (old, advantages, ref, tg), offsets = self._prepare(logits, labels, offsets)
        logp, _ = _logprobs(lg, desc.tokens, tg, vocab, self.scale, self.ignore_index, keep=False)
        loss, self.stats = torch.empty((), dtype=torch.float32, device=lg.device), torch.empty(2, dtype=torch.float32, device=lg.device)
        return L.policy_loss(desc, logp, old, advantages, ref, tg, offsets, loss, self.stats, torch.empty_like(logp))

    def loss_and_grad(self, logits, labels, *, offsets=None, out=None, grad_scale=1.0):
        """(loss, stats, gradient of the logits times ``grad_scale``) without autograd; ``out`` receives the gradient (the logits
        themselves are allowed)."""
        lg, *rest = self._prepare(logits, labels, offsets)
        d, grad = _gradient_buffer(logits, out)
        return self._both(lg, *rest, d, grad_scale), self.stats, grad


# ----------------------------------------------------------------------------------- gradient norm
def _dense(t):
    """Whether a tensor fills its memory without gaps, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != want:
            return False
        want *= size
    return True


_dtype_of = operator.attrgetter("dtype")


_needs_grad = operator.attrgetter("requires_grad")


def _gradient_of(t):
    """The gradient of a parameter (``main_grad`` of an arena's, else ``grad``), another tensor as it is.  A leaf that requires a gradient is a
    parameter whatever its class; a gradient with a graph of its own (create_graph) is no leaf."""
    if isinstance(t, nn.Parameter) or (t.requires_grad and t.is_leaf):
        main = getattr(t, "main_grad", None)
        return t.grad if main is None else main
    return t


def _gradients(tensors):
    """(tensors for the kernels, [(gradient, its copy without gaps)], bb_grad_tensor fields) of a list, empty tensors left out.  (The list is
    gone through property by property: 60 ns each.)"""
    grads = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if set(map(type, grads)) != {torch.Tensor} or any(map(_needs_grad, grads)):
        grads = [t for t in map(_gradient_of, grads) if t is not None]
    sizes = list(map(torch.Tensor.numel, grads))
    if not all(sizes):
        grads, sizes = [t for t, n in zip(grads, sizes) if n], [n for n in sizes if n]
    staged = []
    devices = list(map(torch.Tensor.get_device, grads))
    for device in set(devices):
        _on_current(grads[devices.index(device)], "gradients")
    if not all(map(torch.Tensor.is_contiguous, grads)):
        for at, t in enumerate(grads):
            if not _dense(t):
                grads[at] = t.detach().contiguous()
                staged.append((t.detach(), grads[at]))
    codes = map(L.dtype_codes().get, map(_dtype_of, grads), itertools.repeat(-1))
    return grads, staged, itertools.chain.from_iterable(zip(map(torch.Tensor.data_ptr, grads), sizes, codes, itertools.repeat(0)))


def grad_sumsq(tensors):
    """Sum of squares over all gradients together (fp64 [1] on their device)."""
    grads, _, fields = _gradients(tensors)
    return L.grad_sumsq(L.grad_tensors(fields, len(grads)), len(grads)).clone()


def global_grad_norm(tensors):
    """2-norm over all gradients together (fp32 scalar on their device); nothing is changed."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not _gradients(tensors)[0]:
        return torch.zeros(())
    return grad_sumsq(tensors).sqrt().float().reshape(())


def clip_grad_norm_(tensors, max_norm):
    """Scale the gradients in place so that their global 2-norm is at most ``max_norm``; returns the norm before (fp32 scalar, device).

    ``tensors``: parameters (leaves that require a gradient), or the gradients themselves (bf16 and fp32 may be mixed).  coefficient = min(1,
    max_norm / (norm + 1e-6)); within the norm nothing is written."""
    if not max_norm > 0:
        raise ValueError(f"max_norm has to be positive, got {max_norm}")
    grads, staged, fields = _gradients(tensors)
    if not grads:
        return torch.zeros(())
    norm = L.grad_clip(L.grad_tensors(fields, len(grads)), len(grads), max_norm, torch.empty((), dtype=torch.float32, device=grads[0].device))
    for gradient, copy in staged:
        gradient.copy_(copy)
    return norm


def adam_step_clipped(master, grad, exp_avg, exp_avg_sq, param_lp, *, max_norm, grad_scale=1.0, sumsq=None, **adam):
    """One Adam step over a flat arena on the gradient clipped to ``max_norm``; returns the norm before clipping (fp32 scalar, device).

    ``grad_scale`` multiplies the gradient first (1/dp averaging), the norm included.  ``sumsq``: sum of squares of the unscaled
    gradients that the norm is over (fp64 [1], device) where it covers more than this arena.  ``adam``: as ``lib.adam_step``."""
    if not max_norm > 0:
        raise ValueError(f"max_norm has to be positive, got {max_norm}")
    for t in (master, grad, exp_avg, exp_avg_sq):
        _on_current(t, "adam_step_clipped")
        if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != master.numel():
            raise L.BambooNativeError("adam_step_clipped: contiguous fp32 CUDA tensors of one size are expected")
    if param_lp is not None and (param_lp.get_device() != master.get_device() or param_lp.dtype != torch.bfloat16 or
                                 not param_lp.is_contiguous() or param_lp.numel() != master.numel()):
        raise L.BambooNativeError("adam_step_clipped: the working copy is contiguous bf16, of the arena's size")
    if sumsq is not None and (sumsq.get_device() != master.get_device() or sumsq.dtype != torch.float64):
        raise L.BambooNativeError("adam_step_clipped: sumsq is fp64, on the arena's device")
    norm = torch.empty((), dtype=torch.float32, device=master.device)
    return L.adam_step_clipped(master, grad, exp_avg, exp_avg_sq, param_lp, grad_scale=grad_scale, sumsq=sumsq, max_norm=max_norm, norm=norm, **adam)

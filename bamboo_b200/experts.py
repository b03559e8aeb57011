"""Mixture of experts: what replaces the MLP of a block by several, of which every token takes a few.

    route           the k best experts of every token, their weights, the order of the rows by expert, and the balance term
    dispatch        token rows in that order, a row for every (token, chosen expert)
    grouped_linear  a linear layer per expert over such rows
    expert_mlp      two of them with a GeLU between
    combine         weighted sum of each token's rows, plus a residual

``layers.ExpertMLPHalf`` is the half block made of them.  Formulas stand beside the kernels' declarations (``include/bamboo_b200.h``), the
kernels in ``csrc/experts.cu`` and ``csrc/grouped_gemm.cu``.  How many rows an expert has stays on the device: nothing synchronises, everything
runs on the current stream, CPU tensors and those of another device are refused, and gradients have no gradient of their own.  Indexes that point
nowhere and offsets that do not ascend set the library's status word (``lib.read_status``) and are left out.  Calls can be captured, backward passes
too, as long as no eager graph over the same leaves lives (autograd makes their gradients wait for that graph's stream).
"""
import functools
from typing import NamedTuple, Optional

import torch

from . import lib as L
from .post_training import _aligned_rows, _on_current, _once_differentiable, _rows, _wants_grad


class Routing(NamedTuple):
    """Where every token's rows are.  Slot s = t * k + j is the j-th choice of token t (the tokens of all leading dimensions counted through).
    ``rows`` and ``slots`` are each other's inverse; -1 put into ``rows`` alone drops a choice: its row then counts for nothing, in gradients too."""
    weights: torch.Tensor                       # [..., k] fp32
    experts: torch.Tensor                       # [..., k] int32, -1 where a token has fewer than k
    rows: torch.Tensor                          # [..., k] int32: place of every slot in the order by expert, -1: none
    slots: torch.Tensor                         # [tokens * k] int32: slot at every place, -1 behind the last
    offsets: torch.Tensor                       # [experts + 1] int32: where every expert's places begin
    balance: Optional[torch.Tensor] = None      # [] fp32: 1 where all experts are used alike, more otherwise


# ----------------------------------------------------------------------------------- arguments
_MOST = 2 ** 31 - 1025          # rows and places are counted in 32 bits
_WIDEST = 2 ** 31 - 4097        # ... and so are a row's values, of which loops look some thousand ahead
_device = torch._C._cuda_getDevice


def _int32(t, name, numel=None):
    if t.dtype is torch.int32 and t.is_cuda and t.get_device() == _device() and t.is_contiguous() and (numel is None or t.numel() == numel):
        return t
    _on_current(t, name)
    if t.is_floating_point():
        raise TypeError(f"{name}: integers expected, got {t.dtype}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: {t.numel()} values for {numel}")
    if t.dtype is not torch.int32:
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _row_matrix(t, name):
    """(tensor, rows, row width, stride between rows) of [..., h]: as it is where rows have unit stride and one distance, else a copy."""
    h = t.shape[-1]
    if 0 < h <= _WIDEST and t.is_contiguous() and t.is_cuda and t.get_device() == _device() and t.dtype in L.dtype_codes():
        return t, t.numel() // h, h, h
    _on_current(t, name)
    if t.dtype not in L.dtype_codes():
        raise L.BambooNativeError(f"{name}: bf16 or fp32 expected, got {t.dtype}")
    if h == 0:
        raise ValueError(f"{name}: rows without values")
    if h > _WIDEST:
        raise ValueError(f"{name}: rows of {h} values, at most {_WIDEST}")
    if t.is_contiguous():
        return t, t.numel() // h, h, h
    t = t.detach().reshape(-1, h)
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < h):
        t = t.contiguous()
    return t, t.shape[0], h, t.stride(0) if t.shape[0] > 1 else h


def _plan(routing, tokens=None):
    """(rows, slots, k, tokens) of a routing, checked against each other."""
    rows = _int32(routing.rows, "rows")
    k, count = rows.shape[-1], rows.numel()
    if count > _MOST:
        raise ValueError(f"a routing of {count} rows, at most {_MOST}")
    slots = _int32(routing.slots, "slots", count)
    if tokens is not None and count != tokens * k:
        raise ValueError(f"a routing of {count // k} tokens for {tokens}")
    return rows, slots, k, count // k


# ----------------------------------------------------------------------------------- routing
@functools.lru_cache(maxsize=256)
def _route_desc(tokens, experts, k, normalize, dtype, cols, ld, max_ctas):
    return L.RouteDesc(tokens=tokens, experts=experts, k=k, normalize=normalize, dtype=dtype, cols=cols, ld=ld, max_ctas=max_ctas)


def _route(logits, k, experts, normalize):
    """(logits for the kernels, descriptor, what bb_route_fwd makes)"""
    if logits.dtype not in L.dtype_codes():
        _on_current(logits, "logits")
        raise L.BambooNativeError(f"logits: bf16 or fp32 expected, got {logits.dtype}")
    if logits.shape[-1] > _WIDEST:
        raise ValueError(f"logits of {logits.shape[-1]} columns, at most {_WIDEST}")
    lg, tokens, n = _rows(logits, experts)
    if n > L.max_experts():
        raise ValueError(f"{n} experts: at most {L.max_experts()}")
    if not 0 < k <= min(n, 32):
        raise ValueError(f"k {k}: from 1 to the number of experts ({n}), at most 32")
    dev, shape = lg.device, (*logits.shape[:-1], k)
    weights = torch.empty(shape, dtype=torch.float32, device=dev)
    experts_out, rows = torch.empty(shape, dtype=torch.int32, device=dev), torch.empty(shape, dtype=torch.int32, device=dev)
    slots = torch.empty(tokens * k, dtype=torch.int32, device=dev)
    make = torch.empty if tokens else torch.zeros
    offsets, balance = make(n + 1, dtype=torch.int32, device=dev), make((), dtype=torch.float32, device=dev)
    if tokens * k > _MOST:
        raise ValueError(f"{tokens} tokens with {k} experts each: at most {_MOST} rows")
    desc = _route_desc(tokens, n, k, int(bool(normalize)), L.dtype_codes()[lg.dtype], lg.shape[-1], L._ld(lg) if tokens else lg.shape[-1], L.GEMM_MAX_CTAS)
    # what the backward pass needs of each softmax, then the shares, then scratch of this call (no buffer that calls share: a captured one keeps its own)
    kept = torch.empty(2 * tokens + n + 1 + L.route_scratch(desc) // 4, dtype=torch.float32, device=dev)
    if tokens:
        L.route_fwd(desc, lg, weights, experts_out, rows, slots, offsets, balance, kept)
    return lg, desc, weights, balance, experts_out, rows, slots, offsets, kept


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, experts, normalize):
        lg, desc, weights, balance, chosen, rows, slots, offsets, kept = _route(logits, k, experts, normalize)
        ctx.args = desc, kept, None if lg is logits else logits.shape
        ctx.save_for_backward(lg, chosen)
        ctx.mark_non_differentiable(chosen, rows, slots, offsets)
        ctx.set_materialize_grads(False)
        return weights, balance, chosen, rows, slots, offsets

    @staticmethod
    @_once_differentiable
    def backward(ctx, d_weights, d_balance, *_):
        lg, chosen = ctx.saved_tensors
        desc, kept, shape = ctx.args
        if d_weights is None and d_balance is None:
            return None, None, None, None
        out = torch.empty(lg.shape, dtype=lg.dtype, device=lg.device)
        if desc.tokens:
            if d_weights is not None and not d_weights.is_contiguous():
                d_weights = d_weights.contiguous()
            L.route_bwd(desc, lg, chosen, kept, d_weights, d_balance, out)
        return out if shape is None else out.view(shape), None, None, None


def route(logits, k, experts=None, *, normalize=True):
    """Routing of every token to its ``k`` best experts by ``logits`` [..., cols] (bf16 or fp32), autograd for ``weights`` and ``balance``.

    ``experts``: real columns, at most 256 (the rest is padding with a zero gradient; None: all).  Ties go to the lower index; an expert with a logit of
    -inf is never chosen, so a token whose logits are all -inf has no rows.  The weights are the softmax over all experts; with ``normalize`` over the
    chosen ones.  ``balance`` = experts * sum of f_e P_e (share of rows, mean probability): times a small coefficient it belongs to the loss."""
    if _wants_grad(logits):
        weights, balance, chosen, rows, slots, offsets = _RouteFn.apply(logits, k, experts, normalize)
    else:
        weights, balance, chosen, rows, slots, offsets = _route(logits, k, experts, normalize)[2:8]
    return Routing(weights, chosen, rows, slots, offsets, balance)


# ----------------------------------------------------------------------------------- rows there and back
def _dispatch(x, rows, slots, k):
    xm, tokens, h, ld = _row_matrix(x, "x")
    out = torch.empty(slots.numel(), h, dtype=x.dtype, device=x.device)
    if slots.numel():
        L.dispatch_rows(xm, ld, slots, k, out, tokens)
    return out


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rows, slots, k):
        ctx.k, ctx.shape = k, x.shape
        ctx.save_for_backward(rows)
        return _dispatch(x, rows, slots, k)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dout):
        (rows,) = ctx.saved_tensors
        d, n, h, ld = _row_matrix(dout, "gradient")
        dx = torch.empty(ctx.shape, dtype=dout.dtype, device=dout.device)
        if n:
            L.combine_rows(d, ld, rows, None, None, 0, ctx.k, dx, n // ctx.k, n, h)
        return dx, None, None, None


def dispatch(x, routing):
    """Rows [tokens * k, h] in the order by expert: each the row of ``x`` [..., h] (bf16 or fp32) whose token chose the expert; zeros behind the last.

    The gradient of a token is the sum over its rows, in the order of its choices, in fp32."""
    rows, slots, k, _ = _plan(routing, x.numel() // x.shape[-1] if x.shape[-1] else None)
    return _DispatchFn.apply(x, rows, slots, k) if _wants_grad(x) else _dispatch(x, rows, slots, k)


def _combine(x, weights, residual, rows, k):
    xm, n, h, ld = _row_matrix(x, "rows")
    tokens = rows.numel() // k
    out = torch.empty((*rows.shape[:-1], h) if residual is None else residual.shape, dtype=x.dtype, device=x.device)
    rm, _, _, ld_r = (None, 0, 0, 0) if residual is None else _row_matrix(residual, "residual")
    if tokens:
        L.combine_rows(xm, ld, rows, weights, rm, ld_r, k, out, tokens, n, h)
    return out


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, residual, rows, slots, k):
        ctx.k, ctx.shape, ctx.like = k, x.shape, weights.shape
        ctx.save_for_backward(x if weights.requires_grad else None, weights, rows, slots)
        return _combine(x, weights, residual, rows, k)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dout):
        x, weights, rows, slots = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        d, tokens, h, ld_d = _row_matrix(dout, "gradient")
        dx = torch.empty(ctx.shape, dtype=dout.dtype, device=dout.device) if need_x else None
        dw = torch.empty(ctx.like, dtype=torch.float32, device=dout.device) if need_w else None
        if tokens and (need_x or need_w):
            xm, _, _, ld = _row_matrix(x, "rows") if need_w else (None, 0, 0, h)
            L.combine_rows_bwd(d, ld_d, xm, ld, rows, slots, weights, ctx.k, dx, dw, tokens, slots.numel(), h)
        return dx, dw, dout if need_r else None, None, None, None


def combine(rows, routing, *, residual=None):
    """``residual`` + the sum of every token's rows times ``routing.weights``, summed in fp32 and rounded once; autograd for all three.

    ``rows`` [tokens * k, h] in the order by expert (bf16 or fp32); the result has the shape of ``residual`` [..., h] where that is given."""
    places, slots, k, tokens = _plan(routing)
    if rows.dim() != 2 or rows.shape[0] != slots.numel():
        raise ValueError(f"rows {tuple(rows.shape)} for {slots.numel()} places")
    weights = routing.weights
    _on_current(weights, "weights")
    if weights.numel() != places.numel():
        raise ValueError(f"weights: {weights.numel()} values for {places.numel()}")
    if weights.dtype is not torch.float32:
        weights = weights.to(torch.float32)
    if not weights.is_contiguous():
        weights = weights.contiguous()
    if residual is not None and (residual.dtype != rows.dtype or residual.shape[-1] != rows.shape[1] or residual.numel() != tokens * rows.shape[1]):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype}: a row of {rows.shape[1]} {rows.dtype} for each of {tokens} tokens is expected")
    if _wants_grad(rows) or _wants_grad(weights) or (residual is not None and _wants_grad(residual)):
        return _CombineFn.apply(rows, weights, residual, places, slots, k)
    return _combine(rows, weights, residual, places, k)


# ----------------------------------------------------------------------------------- products
def _weight(w, name, x, transposed=False):
    _on_current(w, name)
    if w.dtype != torch.bfloat16:
        raise L.BambooNativeError(f"{name}: bf16 expected, got {w.dtype}")
    if w.dim() != 3:
        raise ValueError(f"{name} {tuple(w.shape)}: [experts, out, in] is expected")
    if not 0 < w.shape[0] <= L.max_experts():
        raise ValueError(f"{name}: {w.shape[0]} experts, 1 to {L.max_experts()} are possible")
    if w.shape[1] == 0 or w.shape[1] % 8 or w.shape[2] == 0 or w.shape[2] % 8:
        raise ValueError(f"{name} {tuple(w.shape)}: sizes that are multiples of 8 are needed (16-byte rows)")
    if w.shape[1] > _WIDEST or w.shape[2] > _WIDEST:
        raise ValueError(f"{name} {tuple(w.shape)}: sizes of at most {_WIDEST}")
    if w.shape[2] != x:
        raise ValueError(f"{name} {tuple(w.shape)} for rows of {x}")
    return w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.detach().clone(memory_format=torch.contiguous_format)


def _bias(b, name, w):
    if b is None:
        return None
    _on_current(b, name)
    if b.dtype != torch.bfloat16:
        raise L.BambooNativeError(f"{name}: bf16 expected, got {b.dtype}")
    if b.shape != w.shape[:2]:
        raise ValueError(f"{name} {tuple(b.shape)} for a weight {tuple(w.shape)}")
    return b if b.is_contiguous() and b.data_ptr() % 16 == 0 else b.detach().clone(memory_format=torch.contiguous_format)


def _grouped_rows(x, name="x"):
    _on_current(x, name)
    if x.dtype != torch.bfloat16:
        raise L.BambooNativeError(f"{name}: bf16 expected, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"{name} {tuple(x.shape)}: [rows, values] is expected")
    if x.shape[0] > _MOST:
        raise ValueError(f"{name}: {x.shape[0]} rows, at most {_MOST}")
    return _aligned_rows(x, x.shape[1])[0]


def _product(mode, x, w, offsets, width, **kw):
    out = torch.empty(x.shape[0], width, dtype=torch.bfloat16, device=x.device)
    if x.shape[0]:
        L.grouped_gemm(mode, x, w, offsets, out, **kw)
    return out


def _arena_gradient(p):
    """``main_grad`` of a parameter, None where it has none; what the kernels add to is contiguous fp32 of the parameter's shape on 16 bytes."""
    main = getattr(p, "main_grad", None)
    if main is not None and (main.dtype != torch.float32 or main.shape != p.shape or main.get_device() != p.get_device() or not main.is_contiguous() or
                             main.data_ptr() % 16):
        raise L.BambooNativeError(f"main_grad {tuple(main.shape)} {main.dtype}: contiguous fp32 like the parameter {tuple(p.shape)} is expected, on 16 bytes")
    return main


def _weight_gradients(dy, x, offsets, weight, bias, need_w, need_b):
    """(gradient of the weight, of the bias) for autograd; where a parameter belongs to an arena, its fp32 ``main_grad`` is added to instead (None)."""
    grads, empty = {}, dy.shape[0] == 0
    places = {}
    for name, p, wanted in (("weight", weight, need_w), ("bias", bias, need_b)):
        main = _arena_gradient(p) if wanted else None
        grads[name] = (torch.zeros if empty else torch.empty)(p.shape, dtype=torch.bfloat16, device=dy.device) if wanted and main is None else None
        places[name] = main
    if need_w and not empty:
        main = places["weight"]
        size = L.grouped_weight_scratch(dy.shape[0], *weight.shape, need_b)
        scratch = torch.empty(size, dtype=torch.uint8, device=dy.device) if size else None
        L.grouped_gemm(L.GROUPED_WEIGHT, dy, x, offsets, grads["weight"] if main is None else main, epilogue=L.EPI_STORE if main is None else L.EPI_ACCUM_F32,
                       bias_grad=grads["bias"], bias_accum=places["bias"], bias_parts=scratch)
    elif need_b and not empty:
        L.grouped_colsum(dy, offsets, bias.shape[0], out=grads["bias"], accum=places["bias"])
    return grads["weight"], grads["bias"]


class _GroupedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets):
        xm, w, b = _grouped_rows(x), _weight(weight, "weight", x.shape[1]), _bias(bias, "bias", weight)
        ctx.parameters = weight, bias
        ctx.save_for_backward(xm, w, offsets)
        return _product(L.GROUPED_ROWS, xm, w, offsets, w.shape[1], epilogue=L.EPI_STORE if b is None else L.EPI_BIAS, bias=b)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = _grouped_rows(dy, "gradient")
        dx = _product(L.GROUPED_INPUT, dy, w, offsets, w.shape[2]) if need_x else None
        dw, db = _weight_gradients(dy, x, offsets, *ctx.parameters, need_w, need_b)
        return dx, dw, db, None


def _offsets(offsets, weight):
    if offsets.dim() != 1 or offsets.numel() != weight.shape[0] + 1:
        raise ValueError(f"offsets {tuple(offsets.shape)}: one more than there are experts ({weight.shape[0]}), 1-D")
    return _int32(offsets, "offsets")


def grouped_linear(x, weight, offsets, bias=None):
    """y[r] = weight[e] @ x[r] (+ bias[e]) for the rows [offsets[e], offsets[e + 1]) of every expert e; rows of no expert are zeros.

    bf16 ``x`` [rows, k], ``weight`` [experts, n, k], ``bias`` [experts, n], n and k multiples of 8; ``offsets`` [experts + 1] integers on the device.
    Autograd for all three; gradients of weight and bias are added to ``main_grad`` where they belong to an arena, like those of the layers."""
    _on_current(x, "x")
    if weight.dim() != 3:
        raise ValueError(f"weight {tuple(weight.shape)}: [experts, out, in] is expected")
    offsets = _offsets(offsets, weight)
    if any(t is not None and _wants_grad(t) for t in (x, weight, bias)):
        return _GroupedLinearFn.apply(x, weight, bias, offsets)
    xm, w, b = _grouped_rows(x), _weight(weight, "weight", x.shape[-1]), _bias(bias, "bias", weight)
    return _product(L.GROUPED_ROWS, xm, w, offsets, w.shape[1], epilogue=L.EPI_STORE if b is None else L.EPI_BIAS, bias=b)


def _mlp_operands(x, w1, b1, w2, b2):
    return (_grouped_rows(x), _weight(w1, "w1", x.shape[-1]), _bias(b1, "b1", w1), _weight(w2, "w2", w1.shape[1]), _bias(b2, "b2", w2))


def _mlp_desc(x, w1, b1, w2, b2, offsets, *gradients):
    return L.ExpertMLPDesc(*x.shape, w1.shape[1], w2.shape[1], w1.shape[0], L.GEMM_MAX_CTAS, offsets.data_ptr(), w1.data_ptr(), b1.data_ptr(), w2.data_ptr(),
                           b2.data_ptr(), *gradients)


def _mlp_forward(x, w1, b1, w2, b2, offsets):
    """(what the backward pass needs, result): pre-activation and activation stand behind one another in one tensor"""
    rows, inner = x.shape[0], w1.shape[1]
    kept = torch.empty(2, rows, inner, dtype=torch.bfloat16, device=x.device)
    y = torch.empty(rows, w2.shape[1], dtype=torch.bfloat16, device=x.device)
    if rows:
        L.expert_mlp_fwd(_mlp_desc(x, w1, b1, w2, b2, offsets), x, kept, y)
    return kept, y


class _ExpertMLPFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, offsets):
        operands = _mlp_operands(x, w1, b1, w2, b2)
        kept, y = _mlp_forward(*operands, offsets)
        ctx.parameters = w1, b1, w2, b2
        ctx.save_for_backward(*operands, offsets, kept)
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        x, w1, b1, w2, b2, offsets, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = _grouped_rows(dy, "gradient")
        rows, dev = x.shape[0], x.device
        grads, to, added = [], [None] * 4, [None] * 4                # gradients for autograd, and addresses: of those, or of arena gradients
        for at, p in enumerate(ctx.parameters):
            g = None
            if need[1 + at]:
                main = _arena_gradient(p)
                if main is None:
                    g = (torch.empty if rows else torch.zeros)(p.shape, dtype=torch.bfloat16, device=dev)
                    to[at] = g.data_ptr()
                else:
                    added[at] = main.data_ptr()
            grads.append(g)
        dx = torch.empty(rows, x.shape[1], dtype=torch.bfloat16, device=dev) if need[0] else None
        if rows:
            inner = w1.shape[1]
            first = need[0] or need[1] or need[2]
            behind = (2 * rows * inner + 255) & ~255 if first else 0         # the gradient of the pre-activation, then scratch of the weight gradients
            size = L.expert_mlp_scratch(rows, x.shape[1], inner, w2.shape[1], w1.shape[0])
            work = torch.empty(behind + size, dtype=torch.uint8, device=dev)
            L.expert_mlp_bwd(_mlp_desc(x, w1, b1, w2, b2, offsets, *to, *added, work.data_ptr() + behind, size), x, kept, dy, work.data_ptr() if first else None, dx)
        return dx, *grads, None


def expert_mlp(x, offsets, w1, b1, w2, b2):
    """Two layers per expert with a tanh GeLU between: grouped_linear(gelu(grouped_linear(x, w1, offsets, b1)), w2, offsets, b2), where the GeLU
    is taken of the unrounded sums and rounded to bf16 (its slope in the backward pass of the rounded ones): operands of the second product, as the gradient of the
    sums is of the first one's, are bf16.  Together with the result's own rounding 0.24 % in the 2-norm (0.17 % with a GeLU kept in 32 bits).

    w1 [experts, inner, k], b1 [experts, inner], w2 [experts, n, inner], b2 [experts, n]; otherwise as ``grouped_linear``."""
    _on_current(x, "x")
    if w1.dim() != 3 or w2.dim() != 3 or w1.shape[0] != w2.shape[0]:
        raise ValueError(f"w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}: [experts, out, in] with one number of experts is expected")
    if b1 is None or b2 is None:
        raise ValueError("expert_mlp takes both biases")
    offsets = _offsets(offsets, w1)
    if any(_wants_grad(t) for t in (x, w1, b1, w2, b2)):
        return _ExpertMLPFn.apply(x, w1, b1, w2, b2, offsets)
    return _mlp_forward(*_mlp_operands(x, w1, b1, w2, b2), offsets)[1]

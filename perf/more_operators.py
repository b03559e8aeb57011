"""The operators of a mixture of experts and of the optimizer step over its parameters as cases that can be timed and compared: routing
of tokens to experts, moving their rows into the experts' order and back, matrix products grouped by expert, and an AdamW step over a list
of tensors with moments in 32 or 8 bits.

``own`` chooses between the framework's calls and a plain form of the same formulas in elementary 32-bit torch operations;
``exact`` states them once more in 64 bits.  A case's ``kind`` names the operator:

    route     ``route``: the k best experts of every token with their weights, the rows' order by expert, the balance term; with
              ``train`` also the gradient of the logits
    dispatch  ``dispatch``: token rows in the experts' order, and the gradient of the tokens
    combine   ``combine``: weighted sum of each token's rows plus a residual, and the gradients of rows and weights
    product   ``grouped_linear``: a linear layer per expert over ragged groups of rows, and its three gradients
    mlp       ``expert_mlp``: two of them with a GeLU between, and the gradients of rows, weights and biases
    adamw     ``adamw_step_`` over a list of tensors, clipped to a global norm where the case says so
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 256                     # values of a tensor that share a scale where moments have 8 bits
BLOCK_TOP = 256.0               # code of a block's largest value
TINY = 2.0 ** -100              # scales up to this hold nothing
# largest listed sizes, which drawn cases stay below
MAX_LOGITS, MAX_MOVED, MAX_MACS, MAX_WEIGHT, MAX_PARAMS = 32768 * 128, 8192 * 4 * 1024, 3 * 8191 * 4096 * 16384, 8 * 4096 * 16384, 150_000_000
ADAM = {"lr": 1e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01, "step": 7}


def listed():
    return [
        # the toy decoder's tokens over eight experts, latency
        {"name": "route_toy", "kind": "route", "tokens": 512, "experts": 8, "cols": 8, "k": 2, "dtype": "bf16", "normalize": True, "masked": False,
         "train": True},
        # a large batch over many small experts, padding tokens masked out, one expert count that pads its columns
        {"name": "route_batch", "kind": "route", "tokens": 32768, "experts": 125, "cols": 128, "k": 8, "dtype": "fp32", "normalize": False,
         "masked": True, "train": True},
        # the toy decoder's rows
        {"name": "dispatch_toy", "kind": "dispatch", "tokens": 512, "hidden": 256, "experts": 8, "k": 2, "dtype": "bf16", "masked": False, "train": True},
        # the headline decoder's micro-batch, every token to four of 64 experts
        {"name": "dispatch_batch", "kind": "dispatch", "tokens": 8192, "hidden": 1024, "experts": 64, "k": 4, "dtype": "bf16", "masked": True,
         "train": True},
        # a few tokens being scored
        {"name": "combine_few", "kind": "combine", "tokens": 7, "hidden": 1024, "experts": 8, "k": 2, "dtype": "bf16", "masked": False, "train": False},
        # the headline decoder's micro-batch, two experts a token
        {"name": "combine_batch", "kind": "combine", "tokens": 8192, "hidden": 1024, "experts": 8, "k": 2, "dtype": "bf16", "masked": False,
         "train": True},
        # the first layer of eight experts for a few tokens: the weights are the work
        {"name": "product_few", "kind": "product", "rows": 14, "outside": 0, "experts": 8, "n": 4096, "inner": 1024, "bias": True, "train": False},
        # the wide decoder's first layer on an odd number of rows, some of them nobody's, all three products
        {"name": "product_wide", "kind": "product", "rows": 8191, "outside": 160, "experts": 8, "n": 16384, "inner": 4096, "bias": True, "train": True},
        # an expert half of the toy decoder
        {"name": "mlp_toy", "kind": "mlp", "rows": 1024, "outside": 0, "experts": 8, "n": 1024, "inner": 256, "bias": True, "train": True},
        # an expert half of the headline decoder, two experts a token
        {"name": "mlp_batch", "kind": "mlp", "rows": 16384, "outside": 0, "experts": 8, "n": 4096, "inner": 1024, "bias": True, "train": True},
        # the toy decoder's parameters, moments in 32 bits
        {"name": "adamw_toy", "kind": "adamw", "tensors": 52, "elements": 3_500_000, "params": "fp32", "grads": "fp32", "bits": 32, "max_norm": 0.0},
        # bf16 parameters of a few expert blocks with 32-bit masters, moments in 8 bits, gradients clipped
        {"name": "adamw_experts", "kind": "adamw", "tensors": 26, "elements": 150_000_000, "params": "bf16", "grads": "bf16", "bits": 8,
         "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) if hi > lo else lo


def draw(rng):
    """One more case: sizes log-uniform over the range of its kind, odd ones among them."""
    kind = rng.choice(["route", "dispatch", "combine", "product", "mlp", "adamw"])
    train = rng.random() < 0.6
    if kind == "adamw":
        params = rng.choice(["bf16", "fp32"])
        return {"kind": kind, "tensors": rng.randint(1, 60), "elements": _log_int(rng, 1000, MAX_PARAMS // 2), "params": params,
                "grads": rng.choice(["fp32", params]), "bits": rng.choice([8, 8, 32]), "max_norm": rng.choice([0.0, 1.0])}
    if kind == "route":
        experts = _log_int(rng, 2, 256)
        return {"kind": kind, "tokens": _log_int(rng, 1, min(65536, MAX_LOGITS // experts)), "experts": experts,
                "cols": experts if rng.random() < 0.5 else (experts + 7) // 8 * 8, "k": min(experts, rng.randint(1, 8)),
                "dtype": rng.choice(["bf16", "fp32"]), "normalize": rng.random() < 0.5, "masked": rng.random() < 0.5, "train": train}
    if kind in ("dispatch", "combine"):
        hidden, k = 8 * _log_int(rng, 8, 512), rng.randint(1, 8)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        return {"kind": kind, "tokens": _log_int(rng, 1, min(16384, MAX_MOVED // (hidden * k * (1 if dtype == "bf16" else 2)))), "hidden": hidden,
                "experts": max(k, _log_int(rng, 2, 256)), "k": k, "dtype": dtype, "masked": rng.random() < 0.5, "train": train}
    experts = _log_int(rng, 1, 64)
    inner = 8 * _log_int(rng, 8, 512)
    n = 8 * _log_int(rng, 8, max(8, min(1024, MAX_WEIGHT // (experts * inner * 8 * (1 if kind == "product" else 2)))))
    rows = _log_int(rng, 1, max(1, min(20000, MAX_MACS // (inner * n * (1 if kind == "product" else 2) * (3 if train else 1)))))
    return {"kind": kind, "rows": rows, "outside": rng.choice([0, rows // 50]), "experts": experts, "n": n, "inner": inner,
            "bias": rng.random() < 0.5 or kind == "mlp", "train": train}


# ----------------------------------------------------------------------------------- geometry
def _groups(case):
    """Rows of every expert, for these sizes: unequal as a router leaves them, one expert in seven without any."""
    n, total = case["experts"], case["rows"] - case["outside"]
    cuts = random.Random(n * 1_000_003 + total)
    weights = [0.0 if i % 7 == 3 else math.exp(cuts.uniform(0.0, 1.5)) for i in range(n)]
    edges = [int(round(total * sum(weights[:i]) / sum(weights))) for i in range(n + 1)]
    return [b - a for a, b in zip(edges, edges[1:])]


def _masked_tokens(case):
    return case["tokens"] // 16 if case["masked"] else 0


def _tensor_sizes(case):
    """A split of the parameters like a decoder's: a few matrices hold nearly all, biases and gains are short."""
    n, total = case["tensors"], case["elements"]
    cuts = random.Random(n * 1_000_003 + total)
    weights = [math.exp(cuts.uniform(0.0, 9.0)) for _ in range(n)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    return [max(1, s - s % 8 + (3 if i % 5 == 4 else 0)) for i, s in enumerate(sizes)]


# ----------------------------------------------------------------------------------- inputs
def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)


def _router_logits(case, gen):
    """Logits of a router in training: some experts liked better than others; masked tokens have none."""
    x = torch.randn(case["tokens"], case["cols"], device=DEVICE, generator=gen) * 1.5 + torch.randn(case["cols"], device=DEVICE, generator=gen)
    x[torch.randperm(case["tokens"], device=DEVICE, generator=gen)[:_masked_tokens(case)]] = -math.inf
    x[:, case["experts"]:] = 0
    return x.to(DTYPES[case["dtype"]])


def _order(experts, count):
    """(rows, slots, offsets) of chosen experts [T, k] (-1: none): where every slot stands in the order by expert, and back."""
    flat = experts.reshape(-1).long()
    order = torch.sort(torch.where(flat < 0, count, flat), stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(flat.numel(), device=flat.device)
    routed = flat >= 0
    rows = torch.where(routed, place, -1).view(experts.shape).int()
    slots = torch.where(routed[order], order, -1).int()
    offsets = (flat[:, None] == torch.arange(count, device=flat.device)).sum(0).cumsum(0)
    return rows, slots, torch.cat([offsets.new_zeros(1), offsets]).int()


def _moment_blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)


def _encode(x, root):
    """(codes, scales): blocks of x in 8 bits.  root: square roots, whose smallest code that is not 0 stands for all that is smaller."""
    blocks = _moment_blocks(x)
    top = blocks.abs().amax(1)
    finite = torch.isfinite(top)
    factor = torch.where(finite & (top > TINY), BLOCK_TOP / top, 0.0)
    codes = (blocks * factor[:, None]).masked_fill(~finite[:, None], 0.0).to(torch.float8_e4m3fn).float()
    if root:
        codes = torch.where((blocks > 0) & (factor > 0)[:, None], torch.clamp(codes, min=2.0 ** -9), codes)
    return codes.view(-1)[:x.numel()].to(torch.float8_e4m3fn), torch.where(finite, top, math.nan)


def _decode(codes, scales):
    blocks = _moment_blocks(codes.float())
    return (blocks * (scales / BLOCK_TOP)[:, None]).view(-1)[:codes.numel()]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    kind, train = case["kind"], case.get("train", False)
    dtype = DTYPES[case.get("dtype", "bf16")]
    if kind == "route":
        state.update(logits=_router_logits(case, gen).requires_grad_(train), dweights=_randn(gen, case["tokens"], case["k"], scale=1e-2),
                     dbalance=torch.full((), 1e-2, device=DEVICE))
    elif kind in ("dispatch", "combine"):
        t, k, h = case["tokens"], case["k"], case["hidden"]
        logits = torch.randn(t, case["experts"], device=DEVICE, generator=gen) + torch.randn(case["experts"], device=DEVICE, generator=gen)
        weights, experts = torch.sort(torch.softmax(logits, 1), dim=1, descending=True, stable=True)
        experts, weights = experts[:, :k].clone(), weights[:, :k].clone()
        gone = torch.randperm(t, device=DEVICE, generator=gen)[:_masked_tokens(case)]
        experts[gone], weights[gone] = -1, 0
        state["weights"], state["experts"] = weights.requires_grad_(train and kind == "combine"), experts.int()
        state["rows"], state["slots"], state["offsets"] = _order(experts, case["experts"])
        if kind == "dispatch":
            state.update(x=_randn(gen, t, h, dtype=dtype).requires_grad_(train), dout=_randn(gen, t * k, h, dtype=dtype))
        else:
            state.update(x=_randn(gen, t * k, h, dtype=dtype).requires_grad_(train), residual=_randn(gen, t, h, dtype=dtype),
                         dout=_randn(gen, t, h, dtype=dtype))
    elif kind in ("product", "mlp"):
        r, e, n, k = case["rows"], case["experts"], case["n"], case["inner"]
        lengths = _groups(case)
        bf = torch.bfloat16
        state.update(lengths=lengths, offsets=torch.tensor([sum(lengths[:i]) for i in range(e + 1)], device=DEVICE, dtype=torch.int32),
                     x=_randn(gen, r, k, dtype=bf).requires_grad_(train),
                     w1=torch.randn(e, n, k, device=DEVICE, dtype=bf, generator=gen).mul_(1 / math.sqrt(k)).requires_grad_(train),
                     b1=_randn(gen, e, n, dtype=bf, scale=0.1).requires_grad_(train) if case["bias"] else None)
        if kind == "mlp":
            state.update(w2=torch.randn(e, k, n, device=DEVICE, dtype=bf, generator=gen).mul_(1 / math.sqrt(n)).requires_grad_(train),
                         b2=_randn(gen, e, k, dtype=bf, scale=0.1).requires_grad_(train))
        state["dout"] = _randn(gen, r, n if kind == "product" else k, dtype=bf, scale=1e-2)
    else:
        sizes = _tensor_sizes(case)
        starts = [sum((s + 15) // 16 * 16 for s in sizes[:i]) for i in range(len(sizes) + 1)]
        blocks = [-(-s // BLOCK) for s in sizes]
        first = [sum(blocks[:i]) for i in range(len(sizes) + 1)]

        def views(flat):
            return [flat[a:a + s] for a, s in zip(starts, sizes)]
        n = starts[-1]
        state["master"] = 0.02 * torch.randn(n, device=DEVICE, generator=gen)
        state["param"] = state["master"].bfloat16() if case["params"] == "bf16" else None
        state["grad"] = torch.randn(n, device=DEVICE, generator=gen).mul_(1e-2).to(DTYPES[case["grads"]])
        m, v = 1e-3 * torch.randn(n, device=DEVICE, generator=gen), 1e-6 * torch.rand(n, device=DEVICE, generator=gen)
        if case["bits"] == 8:
            state["exp_avg"], state["exp_avg_sq"] = (torch.zeros(n, device=DEVICE, dtype=torch.float8_e4m3fn) for _ in range(2))
            state["scales"] = torch.zeros(2 * first[-1], device=DEVICE)
            for (a, b), (x, y), s in zip(zip(views(state["exp_avg"]), views(state["exp_avg_sq"])), zip(views(m), views(v)),
                                         [state["scales"][2 * i:2 * j].view(2, -1) for i, j in zip(first, first[1:])]):
                for to, value, scale, root in ((a, x, s[0], False), (b, y.sqrt(), s[1], True)):
                    codes, top = _encode(value, root)
                    to.copy_(codes)
                    scale.copy_(top)
        else:
            state["exp_avg"], state["exp_avg_sq"], state["scales"] = m, v, None
        lists = {"masters": "master", "params": "param", "grads": "grad", "exp_avgs": "exp_avg", "exp_avg_sqs": "exp_avg_sq"}
        state.update({k: None if state[f] is None else views(state[f]) for k, f in lists.items()})
        state["scale_list"] = None if state["scales"] is None else [state["scales"][2 * i:2 * j].view(2, -1) for i, j in zip(first, first[1:])]
        if state["params"] is None:
            state["params"], state["masters"] = state["masters"], None
    return state


# ----------------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(state, case):
    kind = case["kind"]
    if kind == "adamw":
        from bamboo_b200 import optim
        norm = optim.adamw_step_(state["params"], state["grads"], state["exp_avgs"], state["exp_avg_sqs"], scales=state["scale_list"],
                                 masters=state["masters"], max_norm=case["max_norm"], **ADAM)
        return ([norm] if case["max_norm"] else []) + _adam_outputs(state)
    from bamboo_b200 import experts as ex
    train = case["train"]
    if kind == "route":
        r = ex.route(state["logits"], case["k"], case["experts"], normalize=case["normalize"])
        grads = torch.autograd.grad((r.weights, r.balance), state["logits"], (state["dweights"], state["dbalance"])) if train else ()
        return [r.weights.detach(), r.experts, r.rows, r.slots, r.offsets, r.balance.detach(), *grads]
    if kind in ("dispatch", "combine"):
        routing = ex.Routing(state["weights"], state["experts"], state["rows"], state["slots"], state["offsets"])
        if kind == "dispatch":
            y, leaves = ex.dispatch(state["x"], routing), (state["x"],)
        else:
            y, leaves = ex.combine(state["x"], routing, residual=state["residual"]), (state["x"], state["weights"])
    elif kind == "product":
        y = ex.grouped_linear(state["x"], state["w1"], state["offsets"], state["b1"])
        leaves = [t for t in (state["x"], state["w1"], state["b1"]) if t is not None]
    else:
        leaves = [state[name] for name in ("x", "w1", "b1", "w2", "b2")]
        y = ex.expert_mlp(state["x"], state["offsets"], *leaves[1:])
    return [y.detach(), *(torch.autograd.grad(y, leaves, state["dout"]) if train else ())]


def _adam_outputs(state):
    return [state[k] for k in ("master", "param", "exp_avg", "exp_avg_sq", "scales") if state[k] is not None]


def _plain_adam(p, master, g, m, v, scales, coef):
    """One tensor's step; moments in 8 bits where there are scales."""
    a = ADAM
    g = g.float() * coef
    m_old, v_old = (m, v) if scales is None else (_decode(m, scales[0]), _decode(v, scales[1]).square())
    m_new = a["beta1"] * m_old + (1 - a["beta1"]) * g
    v_new = a["beta2"] * v_old + (1 - a["beta2"]) * g * g
    w = p if master is None else master
    update = (m_new / (1 - a["beta1"] ** a["step"])) / (torch.sqrt(v_new / (1 - a["beta2"] ** a["step"])) + a["eps"])
    w.copy_(w - a["lr"] * (update + a["weight_decay"] * w))
    if master is not None:
        p.copy_(master)
    if scales is None:
        m.copy_(m_new)
        v.copy_(v_new)
        return
    codes, top = _encode(m_new, False)
    m.copy_(codes)
    scales[0].copy_(top)
    codes, top = _encode(torch.sqrt(v_new), True)
    v.copy_(codes)
    scales[1].copy_(top)


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


def _gelu_slope(x):
    t = torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * x * x)


def _per_expert(state, xs, fn, rest):
    """fn(expert, its rows of every tensor in xs), one behind the other; zeros for rows outside all experts."""
    parts = [fn(e, *part) for e, part in enumerate(zip(*(x[:sum(state["lengths"])].split(state["lengths"]) for x in xs)))]
    return torch.nn.functional.pad(torch.cat(parts), (0, 0, 0, rest))


def _stacked(state, xs, fn):
    return torch.stack([fn(*part) for part in zip(*(x[:sum(state["lengths"])].split(state["lengths"]) for x in xs))])


def _linear(state, x, w, b, rest):
    return _per_expert(state, [x], lambda e, r: r @ w[e].float().t() + (0 if b is None else b[e].float()), rest)


def _linear_gradients(state, dy, x, w, b, rest):
    """(dx, dw, db) in 32 bits"""
    return (_per_expert(state, [dy], lambda e, r: r @ w[e].float(), rest), _stacked(state, [dy, x], lambda d, r: d.t() @ r),
            None if b is None else _stacked(state, [dy], lambda d: d.sum(0)))


def _run_plain(state, case):
    kind = case["kind"]
    if kind == "adamw":
        norm = coef = None
        if case["max_norm"]:
            norm = torch.sqrt(torch.stack([(g.float() * g.float()).sum() for g in state["grads"]]).sum())
            coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
        none = [None] * len(state["grads"])
        [_plain_adam(*each, 1.0 if coef is None else coef) for each in zip(state["params"], state["masters"] or none, state["grads"], state["exp_avgs"],
                                                                           state["exp_avg_sqs"], state["scale_list"] or none)]
        return ([] if norm is None else [norm]) + _adam_outputs(state)
    train = case["train"]
    if kind == "route":
        return _plain_route(state, case)
    if kind == "dispatch":
        x, rows, slots = state["x"].detach(), state["rows"].long(), state["slots"].long()
        y = torch.where((slots >= 0)[:, None], x[torch.clamp(slots, min=0) // case["k"]], 0)
        if not train:
            return [y]
        d = torch.where((rows >= 0)[:, :, None], state["dout"].float()[torch.clamp(rows, min=0)], 0.0)
        return [y, d.sum(1).to(x.dtype)]
    if kind == "combine":
        xs, weights, rows, slots = state["x"].detach(), state["weights"].detach(), state["rows"].long(), state["slots"].long()
        routed = rows >= 0
        each = torch.where(routed[:, :, None], xs.float()[torch.clamp(rows, min=0)], 0.0)
        y = ((weights[:, :, None] * each).sum(1) + state["residual"].float()).to(xs.dtype)
        if not train:
            return [y]
        dy, at = state["dout"].float(), torch.clamp(slots, min=0)
        dxs = torch.where((slots >= 0)[:, None], weights.reshape(-1)[at][:, None] * dy[at // case["k"]], 0.0)
        return [y, dxs.to(xs.dtype), torch.where(routed, (each * dy[:, None]).sum(2), 0.0)]
    x, w1, b1 = (None if state[k] is None else state[k].detach() for k in ("x", "w1", "b1"))
    x, bf, rest = x.float(), torch.bfloat16, case["outside"]
    pre = _linear(state, x, w1, b1, rest)
    if kind == "product":
        if not train:
            return [pre.to(bf)]
        grads = _linear_gradients(state, state["dout"].float(), x, w1, b1, rest)
        return [pre.to(bf), *(g.to(bf) for g in grads if g is not None)]
    w2, b2 = state["w2"].detach(), state["b2"].detach()
    act = _gelu(pre)
    y = _linear(state, act, w2, b2, rest)
    if not train:
        return [y.to(bf)]
    dact, dw2, db2 = _linear_gradients(state, state["dout"].float(), act, w2, b2, rest)
    dx, dw1, db1 = _linear_gradients(state, dact * _gelu_slope(pre), x, w1, b1, rest)
    return [t.to(bf) for t in (y, dx, dw1, db1, dw2, db2)]


def _plain_route(state, case):
    logits, n, k = state["logits"].detach(), case["experts"], case["k"]
    x = logits[:, :n].float()
    value, experts = torch.sort(x, dim=1, descending=True, stable=True)
    value, experts = value[:, :k], experts[:, :k]
    chosen = value > -math.inf
    some = chosen[:, :1]
    e = torch.exp(x - torch.where(some, value[:, :1], 0.0))
    probs = torch.where(some, e / e.sum(1, keepdim=True), 0.0)
    picked = torch.where(chosen, probs.gather(1, experts), 0.0)
    weights = picked
    if case["normalize"]:
        top = torch.where(chosen, torch.exp(value - torch.where(some, value[:, :1], 0.0)), 0.0)
        weights = torch.where(some, top / top.sum(1, keepdim=True), 0.0)
    experts = torch.where(chosen, experts, -1).int()
    rows, slots, offsets = _order(experts, n)
    routed = torch.clamp(some.sum(), min=1).float()
    share = (offsets[1:] - offsets[:-1]).float() / torch.clamp(offsets[-1], min=1).float()
    balance = n * (share * probs.sum(0) / routed).sum()
    out = [weights, experts, rows, slots, offsets, balance]
    if not case["train"]:
        return out
    dw = torch.where(chosen, state["dweights"], 0.0)
    push = state["dbalance"] * n * share / routed
    d = probs * (push - (probs * push).sum(1, keepdim=True))
    mean = (weights * dw).sum(1, keepdim=True)
    if case["normalize"]:
        d = d.scatter_add(1, torch.clamp(experts, min=0).long(), weights * (dw - mean))
    else:
        d = (d - probs * mean).scatter_add(1, torch.clamp(experts, min=0).long(), weights * dw)
    full = torch.zeros(logits.shape, device=d.device, dtype=logits.dtype)
    full[:, :n] = d.to(logits.dtype)
    return out + [full]


# ----------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    kind, train = case["kind"], case.get("train", False)
    if kind == "adamw":
        return _exact_adam(state, case)
    if kind == "route":
        return _exact_route(state, case)
    if kind in ("dispatch", "combine"):
        k, t, rows = case["k"], case["tokens"], state["rows"].long()
        x, dout = state["x"].detach().double(), state["dout"].double()
        place = rows.reshape(-1)
        token = torch.arange(t, device=DEVICE).repeat_interleave(k)[place >= 0]
        slot = torch.arange(t * k, device=DEVICE)[place >= 0]
        place = place[place >= 0]
        if kind == "dispatch":
            y = x.new_zeros(t * k, x.shape[1]).index_copy_(0, place, x[token])
            return [y, torch.zeros_like(x).index_add_(0, token, dout[place])] if train else [y]
        w = state["weights"].detach().double().reshape(-1)
        y = state["residual"].double().index_add_(0, token, w[slot, None] * x[place])
        if not train:
            return [y]
        dw = torch.zeros_like(w).index_copy_(0, slot, torch.einsum("ij,ij->i", dout[token], x[place]))
        return [y, torch.zeros_like(x).index_copy_(0, place, w[slot, None] * dout[token]), dw.view(t, k)]
    x, dout, offsets = state["x"].detach().double(), state["dout"].double(), state["offsets"].tolist()
    names = [n for n in ("w1", "b1", "w2", "b2") if state.get(n) is not None]
    y, dx = torch.zeros_like(dout), torch.zeros_like(x)
    grads = {n: torch.zeros(state[n].shape, dtype=torch.float32, device=DEVICE) for n in names} if train else {}
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if a == b:
            continue
        here = [x[a:b].clone().requires_grad_(train)] + [state[n][e].detach().double().requires_grad_(train) for n in names]
        p = dict(zip(names, here[1:]))
        z = torch.nn.functional.linear(here[0], p["w1"], p.get("b1"))
        if kind == "mlp":
            z = torch.nn.functional.linear(torch.nn.functional.gelu(z, approximate="tanh"), p["w2"], p["b2"])
        y[a:b] = z.detach()
        if train:
            got = torch.autograd.grad(z, here, dout[a:b])
            dx[a:b] = got[0]
            for n, g in zip(names, got[1:]):
                grads[n][e] = g
    return [y, dx, *grads.values()] if train else [y]


def _exact_route(state, case):
    n, k, t = case["experts"], case["k"], case["tokens"]
    x = state["logits"].detach()[:, :n].double().requires_grad_(True)
    left, picks = x.detach().clone(), []
    for _ in range(k):
        best = left.argmax(1)
        picks.append(torch.where(left.amax(1) > -math.inf, best, -1))
        left.scatter_(1, best[:, None], -math.inf)
    experts = torch.stack(picks, 1)
    alive = experts[:, 0] >= 0
    member = torch.zeros(t, n + 1, dtype=torch.bool, device=DEVICE).scatter_(1, torch.where(experts < 0, n, experts), True)[:, :n]
    probs = torch.zeros_like(x).index_put((alive.nonzero()[:, 0],), torch.softmax(x[alive], 1))
    base = probs
    if case["normalize"]:
        base = torch.zeros_like(x).index_put((alive.nonzero()[:, 0],), torch.softmax(x.masked_fill(~member, -math.inf)[alive], 1))
    weights = base.gather(1, experts.clamp(min=0)) * (experts >= 0)
    count = member.sum(0).double()
    balance = n * torch.dot(count / count.sum().clamp(min=1), probs.sum(0) / alive.sum().clamp(min=1))
    rows, slots, offsets = _order(experts, n)
    out = [weights.detach(), experts.int(), rows, slots, offsets, balance.detach()]
    if not case["train"]:
        return out
    (dx,) = torch.autograd.grad((weights, balance), x, (state["dweights"].double(), state["dbalance"].double()))
    return out + [torch.nn.functional.pad(dx, (0, case["cols"] - n))]


def _exact_adam(state, case):
    b1, b2, step = ADAM["beta1"], ADAM["beta2"], ADAM["step"]
    grad = torch.zeros(state["grad"].shape, dtype=torch.float64, device=DEVICE)     # (nothing between the tensors)
    for to, g in zip(torch.split(grad, [(s + 15) // 16 * 16 for s in _tensor_sizes(case)]), state["grads"]):
        to[:g.numel()] = g.double()
    norm = torch.linalg.vector_norm(grad)
    if case["max_norm"]:
        grad *= min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    p = state["master"].double()
    eight = case["bits"] == 8
    if eight:
        spread = torch.zeros(2, *grad.shape, dtype=torch.float64, device=DEVICE)
        at = 0
        for g, s in zip(state["grads"], state["scale_list"]):
            n = g.numel()
            spread[:, at:at + n] = s.double().repeat_interleave(BLOCK, 1)[:, :n] / BLOCK_TOP
            at += (n + 15) // 16 * 16
        m, v = state["exp_avg"].double() * spread[0], (state["exp_avg_sq"].double() * spread[1]).square()
    else:
        m, v = state["exp_avg"].double(), state["exp_avg_sq"].double()
    m, v = torch.lerp(grad, m, b1), torch.lerp(grad.square(), v, b2)
    new = p * (1 - ADAM["lr"] * ADAM["weight_decay"]) - ADAM["lr"] * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + ADAM["eps"])
    scales = None
    at = 0
    if eight:
        scales = []
    for g in state["grads"]:                                                        # what stands between the tensors stays
        n, end = g.numel(), at + (g.numel() + 15) // 16 * 16
        new[at + n:end] = p[at + n:end]
        if eight:
            scales += [_moment_blocks(m[at:at + n]).abs().amax(1), _moment_blocks(v[at:at + n].sqrt()).amax(1)]
        else:
            m[at + n:end], v[at + n:end] = state["exp_avg"][at + n:end].double(), state["exp_avg_sq"][at + n:end].double()
        at = end
    out = [norm] if case["max_norm"] else []
    out += [new] + ([new] if state["param"] is not None else [])
    return out + ([None, None, torch.cat(scales)] if eight else [m, v])


# ----------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, train = case["kind"], case.get("train", False)
    item = 2 if case.get("dtype", "bf16") == "bf16" else 4
    if kind == "adamw":
        n = sum(_tensor_sizes(case))
        grad = 2 if case["grads"] == "bf16" else 4
        return {"bytes": n * (8 + grad + (2 if case["params"] == "bf16" else 0) + (4 if case["bits"] == 8 else 16)), "flops": 17 * n}
    if kind == "route":
        t, n, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": t * (n * item + 16 * k) + (t * (case["cols"] * item + 4 * k) if train else 0), "flops": t * n * (4 + k + (6 if train else 0))}
    if kind in ("dispatch", "combine"):
        t, k, h = case["tokens"] - _masked_tokens(case), case["k"], case["hidden"]
        small = case["tokens"] * h * item
        large = case["tokens"] * k * h * item                # rows that are written are written for masked tokens too
        if kind == "dispatch":
            return {"bytes": small + large + (t * k * h * item + small if train else 0), "flops": t * k * h if train else t * k}
        return {"bytes": t * k * h * item + 2 * small + (large + small if train else 0), "flops": t * k * h * (6 if train else 2)}
    groups = _groups(case)
    rows, used, n, k = sum(groups), sum(g > 0 for g in groups), case["n"], case["inner"]
    matrices, wide = (2, 0) if kind == "mlp" else (1, case["rows"] * n)
    narrow = case["rows"] * k * (2 if kind == "mlp" else 1)
    size = 2 * (narrow + wide + matrices * used * n * k)
    flops = 2 * matrices * rows * n * k
    if train:       # what arrives, the gradient of the rows, and that of every expert's weights, those without rows too
        size += 2 * (narrow + wide + matrices * case["experts"] * n * k)
        flops *= 3
    return {"bytes": size, "flops": flops}

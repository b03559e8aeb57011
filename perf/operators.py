"""The operators of a post-training step as cases that can be timed and compared: log-probabilities of given tokens with their
gradient (from logits, and from hidden states through the vocabulary projection), the paired preference loss and the clipped
policy loss over them, the global gradient norm with clipping, and the Adam step that clips.

``own`` chooses between the framework's calls and a plain form of the same formulas in elementary 32-bit torch operations;
``exact`` states them once more in 64 bits.  A case's ``kind`` names the operator:

    logprob     ``token_logprobs``: forward, or forward and gradient of the logits
    head        ``head_logprobs``: forward, or forward and gradients of hidden states and weight
    preference  ``PreferenceLoss.loss_and_grad``: loss, rewards and gradient of the logits
    policy      ``PolicyLoss.loss_and_grad``: loss, statistics and gradient of the logits
    clip        ``clip_grad_norm_`` over a list of gradients
    step        ``adam_step_clipped`` over a flat parameter arena
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# largest listed sizes, which drawn cases stay below
MAX_LOGITS, MAX_HEAD, MAX_GRADS, MAX_PARAMS = 8192 * 50257, 4096 * 50257 * 1024, 160_000_000, 120_000_000
ADAM = {"lr": 1e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01, "step": 7}


def listed():
    return [
        # scoring what a few sequences answered last: one row each, nothing to learn; fp32 logits without padding
        {"name": "score_few_rows", "kind": "logprob", "rows": 3, "vocab": 50257, "cols": 50257, "dtype": "fp32", "train": False,
         "temperature": 0.7},
        # the headline decoder's micro-batch: 8 sequences of 1024 tokens, padded vocabulary
        {"name": "logprob_train", "kind": "logprob", "rows": 8192, "vocab": 50257, "cols": 50304, "dtype": "bf16", "train": True,
         "temperature": 1.0},
        # a reference model's last layer on a ragged number of tokens (the vocabulary head of the layer benchmark)
        {"name": "head_score", "kind": "head", "rows": 999, "hidden": 1024, "vocab": 50257, "cols": 50304, "train": False,
         "temperature": 1.0},
        # the policy's last layer on half a micro-batch, gradients of hidden states and weight included
        {"name": "head_train", "kind": "head", "rows": 4096, "hidden": 1024, "vocab": 50257, "cols": 50304, "train": True,
         "temperature": 1.0},
        # the toy decoder that a user tries the loss with: two pairs of 128 tokens, latency
        {"name": "preference_toy", "kind": "preference", "sequences": 4, "tokens": 512, "ragged": False, "vocab": 1024, "cols": 1024,
         "dtype": "bf16", "temperature": 1.0, "form": "sigmoid", "smoothing": 0.0, "average": False, "beta": 0.1},
        # two pairs at the headline decoder's length, prompts masked
        {"name": "preference_pairs", "kind": "preference", "sequences": 4, "tokens": 4096, "ragged": False, "vocab": 50257,
         "cols": 50304, "dtype": "bf16", "temperature": 1.0, "form": "sigmoid", "smoothing": 0.1, "average": False, "beta": 0.1},
        # one micro-batch of the toy decoder under the policy loss, latency
        {"name": "policy_toy", "kind": "policy", "sequences": 4, "tokens": 512, "ragged": False, "vocab": 1024, "cols": 1024,
         "dtype": "bf16", "temperature": 1.0, "reduction": "token", "kl": 0.05, "reference": True},
        # sampled answers of unequal lengths packed behind one another, 16 of them, the headline decoder's vocabulary
        {"name": "policy_packed", "kind": "policy", "sequences": 16, "tokens": 7777, "ragged": True, "vocab": 50257, "cols": 50304,
         "dtype": "bf16", "temperature": 0.8, "reduction": "sequence", "kl": 0.05, "reference": True},
        # the toy decoder's gradients, a tensor for each parameter
        {"name": "clip_toy", "kind": "clip", "tensors": 52, "elements": 3_500_000, "dtype": "fp32", "max_norm": 1.0},
        # four blocks and the vocabulary matrices of the headline decoder in bf16
        {"name": "clip_blocks", "kind": "clip", "tensors": 52, "elements": 153_000_000, "dtype": "bf16", "max_norm": 1.0},
        # one arena of the toy decoder
        {"name": "step_toy", "kind": "step", "elements": 3_500_000, "max_norm": 1.0},
        # a pipeline stage of the headline decoder: four blocks and the embedding
        {"name": "step_stage", "kind": "step", "elements": 102_900_000, "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the range of its kind, odd ones among them."""
    kind = rng.choice(["logprob", "head", "preference", "policy", "clip", "step"])
    vocab = _log_int(rng, 200, 51000)
    cols = vocab if rng.random() < 0.3 else (vocab + 127) // 128 * 128
    temperature = rng.choice([1.0, 1.0, 0.7, 1.3])
    if kind == "head":
        hidden = 8 * _log_int(rng, 8, 256)
        rows = _log_int(rng, 1, max(1, min(8192, MAX_HEAD // (vocab * hidden))))
        return {"kind": kind, "rows": rows, "hidden": hidden, "vocab": vocab, "cols": cols, "train": rng.random() < 0.5,
                "temperature": temperature}
    if kind == "clip":
        return {"kind": kind, "tensors": rng.randint(1, 60), "elements": _log_int(rng, 1000, MAX_GRADS // 2),
                "dtype": rng.choice(["fp32", "bf16", "mixed"]), "max_norm": rng.choice([0.5, 1.0, 5.0])}
    if kind == "step":
        return {"kind": kind, "elements": _log_int(rng, 1000, MAX_PARAMS), "max_norm": rng.choice([0.5, 1.0, 5.0])}
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    most = min(16384, MAX_LOGITS // (vocab * (1 if dtype == "bf16" else 2)))
    if kind == "logprob":
        return {"kind": kind, "rows": _log_int(rng, 1, most), "vocab": vocab, "cols": cols, "dtype": dtype,
                "train": rng.random() < 0.6, "temperature": temperature}
    sequences = 2 * rng.randint(1, 8)
    length = _log_int(rng, 1, max(1, most // sequences))
    ragged = rng.random() < 0.5
    case = {"kind": kind, "sequences": sequences, "tokens": length * sequences + (rng.randrange(sequences) if ragged else 0),
            "ragged": ragged, "vocab": vocab, "cols": cols, "dtype": dtype, "temperature": temperature}
    if kind == "preference":
        case.update(form=rng.choice(["sigmoid", "sigmoid", "squared"]), smoothing=rng.choice([0.0, 0.1]),
                    average=rng.random() < 0.3, beta=rng.choice([0.1, 0.3]))
    else:
        case.update(reduction=rng.choice(["token", "sequence"]), kl=rng.choice([0.0, 0.05]), reference=True)
        case["reference"] = case["kl"] > 0
    return case


# ----------------------------------------------------------------------------------- geometry
def _lengths(case):
    """Tokens of each sequence: equal, or (ragged) a fixed split of the total for these sizes."""
    n, total = case["sequences"], case["tokens"]
    if not case["ragged"]:
        return [total // n] * n
    cuts = random.Random(n * 1_000_003 + total)
    marks = sorted(cuts.randrange(total + 1) for _ in range(n - 1))
    return [b - a for a, b in zip([0] + marks, marks + [total])]


def _prompt(i, length):
    """Leading tokens of sequence i that are a prompt and do not count: up to two fifths of it."""
    return (i * 7 + 3) % 11 * length * 2 // 50


def _counted_rows(case):
    if case["kind"] in ("logprob", "head"):
        return case["rows"] - case["rows"] // 16
    return sum(n - _prompt(i, n) for i, n in enumerate(_lengths(case)))


def _tensor_sizes(case):
    """A split of the gradients like a decoder's: a few matrices hold nearly all, biases and gains are short."""
    n, total = case["tensors"], case["elements"]
    cuts = random.Random(n * 1_000_003 + total)
    weights = [math.exp(cuts.uniform(0.0, 9.0)) for _ in range(n)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    return [max(1, s - s % 8 + (3 if i % 5 == 4 else 0)) for i, s in enumerate(sizes)]


def _grad_dtype(case, i):
    return torch.bfloat16 if case["dtype"] == "bf16" or (case["dtype"] == "mixed" and i % 2) else torch.float32


# ----------------------------------------------------------------------------------- inputs
def _logits_and_targets(case, rows, gen):
    """Logits as a trained model's: a spread of a few units, the target among the likely ones half of the time, zero where
    columns only pad the vocabulary."""
    dtype, vocab, cols = DTYPES[case["dtype"]], case["vocab"], case["cols"]
    logits = torch.randn(rows, cols, device=DEVICE, dtype=dtype, generator=gen).mul_(2.0)
    logits[:, vocab:] = 0
    targets = torch.randint(0, vocab, (rows,), device=DEVICE, generator=gen)
    index = torch.arange(rows, device=DEVICE)
    likely = torch.rand(rows, device=DEVICE, generator=gen) < 0.5
    logits[index, targets] += torch.where(likely, 8.0, 0.0).to(dtype)
    return logits, targets


def _sampled_logps(logits, targets, case):
    x = logits[:, :case["vocab"]].float() / case["temperature"]
    return x.gather(1, targets[:, None])[:, 0] - torch.logsumexp(x, 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    kind = case["kind"]
    if kind == "logprob":
        logits, targets = _logits_and_targets(case, case["rows"], gen)
        targets[torch.randperm(case["rows"], device=DEVICE, generator=gen)[:case["rows"] // 16]] = IGNORE
        state.update(logits=logits.requires_grad_(case["train"]), targets=targets,
                     grad=torch.randn(case["rows"], device=DEVICE, generator=gen) / case["rows"])
    elif kind == "head":
        # hidden states behind a LayerNorm, weights at their initial spread
        hidden = torch.randn(case["rows"], case["hidden"], device=DEVICE, generator=gen).bfloat16()
        weight = (torch.randn(case["cols"], case["hidden"], device=DEVICE, generator=gen) * 1.5 / math.sqrt(case["hidden"])).bfloat16()
        weight[case["vocab"]:] = 0
        targets = torch.randint(0, case["vocab"], (case["rows"],), device=DEVICE, generator=gen)
        targets[torch.randperm(case["rows"], device=DEVICE, generator=gen)[:case["rows"] // 16]] = IGNORE
        state.update(hidden=hidden.requires_grad_(case["train"]), weight=weight.requires_grad_(case["train"]), targets=targets,
                     grad=torch.randn(case["rows"], device=DEVICE, generator=gen) / case["rows"])
    elif kind in ("preference", "policy"):
        lengths = _lengths(case)
        logits, targets = _logits_and_targets(case, case["tokens"], gen)
        logps = _sampled_logps(logits, targets, case)
        starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        counts = torch.ones(case["tokens"], dtype=torch.bool)
        for i, n in enumerate(lengths):
            counts[starts[i]:starts[i] + _prompt(i, n)] = False
        targets = torch.where(counts.to(DEVICE), targets, IGNORE)
        noise = torch.randn(case["tokens"], device=DEVICE, generator=gen)
        state.update(logits=logits, offsets=torch.tensor(starts, device=DEVICE) if case["ragged"] else None,
                     counts=counts, lengths=lengths, reference=logps + 0.1 * noise)
        if kind == "policy":
            # how far the policy moved since it sampled; nothing within a few thousandths of the clipping bounds, where the
            # gradient jumps and 32 bits cannot say on which side a token is
            moved = 0.15 * torch.randn(case["tokens"], device=DEVICE, generator=gen)
            for bound in (math.log(0.8), math.log(1.2)):
                moved = torch.where((moved - bound).abs() < 2e-3, moved + 8e-3, moved)
            state.update(old=logps - moved, advantages=torch.randn(case["tokens"], device=DEVICE, generator=gen) + 0.3)
            if not case["reference"]:
                state["reference"] = None
        shape = (case["tokens"],) if case["ragged"] else (case["sequences"], case["tokens"] // case["sequences"])
        state["logits"] = state["logits"].view(*shape, case["cols"])
        state["targets"] = targets.view(shape)
        state.update({k: state[k].view(shape) for k in ("reference", "old", "advantages") if state.get(k) is not None})
    elif kind == "clip":
        state["grads"] = [(0.02 * torch.randn(n, device=DEVICE, generator=gen)).to(_grad_dtype(case, i))
                          for i, n in enumerate(_tensor_sizes(case))]
    else:
        n = (case["elements"] + 7) // 8 * 8
        state["master"] = 0.02 * torch.randn(n, device=DEVICE, generator=gen)
        state["grad"] = 1e-2 * torch.randn(n, device=DEVICE, generator=gen)
        state["exp_avg"] = 1e-3 * torch.randn(n, device=DEVICE, generator=gen)
        state["exp_avg_sq"] = 1e-6 * torch.rand(n, device=DEVICE, generator=gen)
        state["lp"] = state["master"].bfloat16()
    return state


# ----------------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(state, case):
    from bamboo_b200 import post_training as pt
    kind = case["kind"]
    if kind == "logprob":
        if not case["train"]:
            return pt.token_logprobs(state["logits"], state["targets"], case["vocab"], temperature=case["temperature"])
        logps = pt.token_logprobs(state["logits"], state["targets"], case["vocab"], temperature=case["temperature"])
        return [logps.detach(), *torch.autograd.grad(logps, state["logits"], state["grad"])]
    if kind == "head":
        logps = pt.head_logprobs(state["hidden"], state["weight"], state["targets"], case["vocab"], temperature=case["temperature"])
        if not case["train"]:
            return logps
        return [logps.detach(), *torch.autograd.grad(logps, (state["hidden"], state["weight"]), state["grad"])]
    if kind == "preference":
        loss_fn = pt.PreferenceLoss(case["vocab"], beta=case["beta"], form=case["form"], label_smoothing=case["smoothing"],
                                    average=case["average"], temperature=case["temperature"])
        return loss_fn.loss_and_grad(state["logits"], (state["targets"], state["reference"]), offsets=state["offsets"])
    if kind == "policy":
        loss_fn = pt.PolicyLoss(case["vocab"], clip_low=0.2, clip_high=0.2, kl_coef=case["kl"], reduction=case["reduction"],
                                temperature=case["temperature"])
        labels = (state["targets"], state["old"], state["advantages"]) + ((state["reference"],) if case["reference"] else ())
        return loss_fn.loss_and_grad(state["logits"], labels, offsets=state["offsets"])
    if kind == "clip":
        return [pt.clip_grad_norm_(state["grads"], case["max_norm"]), *state["grads"]]
    norm = pt.adam_step_clipped(state["master"], state["grad"], state["exp_avg"], state["exp_avg_sq"], state["lp"],
                                max_norm=case["max_norm"], **ADAM)
    return [norm, state["master"], state["exp_avg"], state["exp_avg_sq"], state["lp"]]


def _plain_logprobs(x, targets):
    """x [rows, V] in 32 bits: log-probabilities of the targets (0 where they do not count), softmax, counted rows."""
    counted = targets != IGNORE
    at = torch.where(counted, targets, 0)[:, None]
    top = x.max(1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    logps = torch.where(counted, (x.gather(1, at) - top - torch.log(total))[:, 0], 0.0)
    return logps, e / total, counted, at


def _plain_dlogits(probs, at, row_grad, temperature, cols, dtype):
    d = probs * -(row_grad / temperature)[:, None]
    d.scatter_add_(1, at, (row_grad / temperature)[:, None])
    out = torch.zeros(d.shape[0], cols, device=d.device, dtype=dtype)
    out[:, :d.shape[1]] = d.to(dtype)
    return out


def _run_plain(state, case):
    kind = case["kind"]
    if kind == "clip":
        norm = torch.sqrt(torch.stack([(g.float() * g.float()).sum() for g in state["grads"]]).sum())
        coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
        return [norm, *[g.copy_(g.float() * coef) for g in state["grads"]]]
    if kind == "step":
        a = ADAM
        grad, m, v, p = state["grad"], state["exp_avg"], state["exp_avg_sq"], state["master"]
        norm = torch.sqrt((grad * grad).sum())
        g = grad * torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
        m.copy_(a["beta1"] * m + (1 - a["beta1"]) * g)
        v.copy_(a["beta2"] * v + (1 - a["beta2"]) * g * g)
        step = (m / (1 - a["beta1"] ** a["step"])) / (torch.sqrt(v / (1 - a["beta2"] ** a["step"])) + a["eps"])
        p.copy_(p - a["lr"] * (step + a["weight_decay"] * p))
        state["lp"].copy_(p)
        grad.zero_()
        return [norm, p, m, v, state["lp"]]
    targets, t = state["targets"].reshape(-1), case["temperature"]
    if kind == "head":
        hidden, weight = state["hidden"].detach().float(), state["weight"].detach()[:case["vocab"]].float()
        logps, probs, counted, at = _plain_logprobs(hidden @ weight.t() / t, targets)
        if not case["train"]:
            return logps
        d = _plain_dlogits(probs, at, torch.where(counted, state["grad"], 0.0), t, case["vocab"], torch.float32)
        dweight = torch.zeros(state["weight"].shape, device=d.device, dtype=torch.bfloat16)
        dweight[:case["vocab"]] = (d.t() @ hidden).bfloat16()
        return [logps, (d @ weight).bfloat16(), dweight]
    logits = state["logits"].detach()
    logps, probs, counted, at = _plain_logprobs(logits.reshape(-1, case["cols"])[:, :case["vocab"]].float() / t, targets)
    if kind == "logprob":
        if not case["train"]:
            return logps
        return [logps, _plain_dlogits(probs, at, torch.where(counted, state["grad"], 0.0), t, case["cols"], logits.dtype)]
    n = case["sequences"]
    lengths = torch.tensor(state["lengths"], device=DEVICE)
    owner = torch.repeat_interleave(torch.arange(n, device=DEVICE), lengths, output_size=case["tokens"])
    count = torch.zeros(n, device=DEVICE).index_add_(0, owner, counted.float())
    if kind == "preference":
        ratio = torch.where(counted, logps - state["reference"].reshape(-1), 0.0)
        length = torch.clamp(count, min=1.0) if case["average"] else torch.ones_like(count)
        score = torch.zeros(n, device=DEVICE).index_add_(0, owner, ratio) / length
        beta, e = case["beta"], case["smoothing"]
        h = beta * (score[0::2] - score[1::2])
        if case["form"] == "sigmoid":
            softplus = lambda z: torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))  # noqa: E731
            each = (1 - e) * softplus(-h) + e * softplus(h)
            slope = -(1 - e) / (1 + torch.exp(h)) + e / (1 + torch.exp(-h))
        else:
            each = (h / beta - 0.5 / beta) ** 2
            slope = 2 * (h / beta - 0.5 / beta) / beta
        push = torch.stack([slope, -slope], 1).reshape(-1) * beta / (n // 2) / length
        grad = torch.where(counted, push[owner], 0.0)
        dlogits = _plain_dlogits(probs, at, grad, t, case["cols"], logits.dtype)
        return [each.mean(), beta * score, dlogits.view(logits.shape)]
    adv = state["advantages"].reshape(-1)
    ratio = torch.exp(torch.where(counted, logps - state["old"].reshape(-1), 0.0))
    bounded = torch.clamp(ratio, 0.8, 1.2)
    clipped = counted & (bounded * adv < ratio * adv)
    each = -torch.minimum(ratio * adv, bounded * adv)
    slope = torch.where(clipped, 0.0, -ratio * adv)
    kl = torch.zeros_like(ratio)
    if case["reference"]:
        gap = torch.where(counted, state["reference"].reshape(-1) - logps, 0.0)
        kl = torch.exp(gap) - gap - 1
        each, slope = each + case["kl"] * kl, slope + case["kl"] * (1 - torch.exp(gap))
    total = torch.clamp(count.sum(), min=1.0)
    weight = 1 / total if case["reduction"] == "token" else (1 / (n * torch.clamp(count, min=1.0)))[owner]
    weight = torch.where(counted, weight, 0.0)
    dlogits = _plain_dlogits(probs, at, slope * weight, t, case["cols"], logits.dtype)
    stats = torch.stack([torch.where(counted, kl, 0.0).sum() / total, clipped.sum() / total])
    return [(torch.where(counted, each, 0.0) * weight).sum(), stats, dlogits.view(logits.shape)]


# ----------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        parts = [g.double() for g in state["grads"]]
        norm = torch.linalg.vector_norm(torch.cat(parts))
        scale = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        return [norm, *[g * scale for g in parts]]
    if kind == "step":
        p, g, m, v = (state[k].double() for k in ("master", "grad", "exp_avg", "exp_avg_sq"))
        norm = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        b1, b2, k = ADAM["beta1"], ADAM["beta2"], ADAM["step"]
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g.square(), v, b2)
        p = p * (1 - ADAM["lr"] * ADAM["weight_decay"]) - ADAM["lr"] * (m / (1 - b1 ** k)) / ((v / (1 - b2 ** k)).sqrt() + ADAM["eps"])
        return [norm, p, m, v, p]
    targets = state["targets"].reshape(-1)
    mask = targets.ne(IGNORE)
    index = targets.clamp(min=0)
    rows = torch.arange(targets.numel(), device=DEVICE)
    if kind == "head":
        h, w = state["hidden"].detach().double(), state["weight"].detach()[:case["vocab"]].double()
        x = torch.mm(h, w.t())
    else:
        x = state["logits"].detach().reshape(targets.numel(), -1)[:, :case["vocab"]].double()
    table = torch.log_softmax(x / case["temperature"], dim=1)
    del x
    logps = table[rows, index] * mask

    def gradient(row_grad):
        """Gradient of sum(row_grad * logps) with respect to the logits."""
        row_grad = row_grad * mask / case["temperature"]
        d = table.exp().mul_(-row_grad[:, None])
        d[rows, index] += row_grad
        return d
    if kind == "head":
        if not case["train"]:
            return logps
        d = gradient(state["grad"].double())
        return [logps, d @ w, torch.nn.functional.pad(d.t() @ h, (0, 0, 0, case["cols"] - case["vocab"]))]
    pad = (0, case["cols"] - case["vocab"])
    if kind == "logprob":
        return [logps, torch.nn.functional.pad(gradient(state["grad"].double()), pad)] if case["train"] else logps
    n, lengths = case["sequences"], state["lengths"]
    member = torch.zeros(n, targets.numel(), dtype=torch.float64, device=DEVICE)       # which tokens count for which sequence
    start = 0
    for i, length in enumerate(lengths):
        member[i, start:start + length] = 1
        start += length
    member *= mask
    counts = member.sum(1)
    if kind == "preference":
        z = (logps - state["reference"].reshape(-1).double()).masked_fill(~mask, 0).requires_grad_(True)
        score = member @ z
        if case["average"]:
            score = score / counts.clamp(min=1)
        rewards = case["beta"] * score
        h = rewards[0::2] - rewards[1::2]
        if case["form"] == "sigmoid":
            logsig = torch.nn.functional.logsigmoid
            loss = (-(1 - case["smoothing"]) * logsig(h) - case["smoothing"] * logsig(-h)).mean()
        else:
            loss = (h / case["beta"] - 1 / (2 * case["beta"])).square().mean()
        (row_grad,) = torch.autograd.grad(loss, z)
        return [loss.detach(), rewards.detach(), torch.nn.functional.pad(gradient(row_grad), pad).view(state["logits"].shape)]
    z = logps.clone().requires_grad_(True)
    adv = state["advantages"].reshape(-1).double()
    ratio = (z - state["old"].reshape(-1).double()).masked_fill(~mask, 0).exp()
    unclipped, bounded = ratio * adv, ratio.clamp(0.8, 1.2) * adv
    each = -torch.where(bounded < unclipped, bounded, unclipped)
    kl = torch.zeros_like(each)
    if case["reference"]:
        gap = (state["reference"].reshape(-1).double() - z).masked_fill(~mask, 0)
        kl = gap.exp() - gap - 1
    each = (each + case["kl"] * kl) * mask
    total = counts.sum().clamp(min=1)
    loss = each.sum() / total if case["reduction"] == "token" else ((member @ each) / counts.clamp(min=1)).mean()
    (row_grad,) = torch.autograd.grad(loss, z)
    stats = torch.stack([(kl.detach() * mask).sum(), ((bounded < unclipped) & mask).sum().double()]) / total
    return [loss.detach(), stats, torch.nn.functional.pad(gradient(row_grad), pad).view(state["logits"].shape)]


# ----------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "clip":
        sizes = _tensor_sizes(case)
        return {"bytes": sum(2 * n * (2 if _grad_dtype(case, i) == torch.bfloat16 else 4) for i, n in enumerate(sizes)),
                "flops": 3 * sum(sizes)}
    if kind == "step":
        # read p, g, m, v; write p, g, m, v in 32 bits and the bf16 copy
        return {"bytes": 34 * case["elements"], "flops": 17 * case["elements"]}
    rows, counted = case["rows"] if kind in ("logprob", "head") else case["tokens"], _counted_rows(case)
    vocab, cols = case["vocab"], case["cols"]
    if kind == "head":
        flops, size = 2 * counted * vocab * case["hidden"], (rows + vocab) * case["hidden"] * 2 + 12 * rows
        if case["train"]:
            flops, size = 3 * flops, size + (rows + cols) * case["hidden"] * 2 + 4 * rows
        return {"bytes": size, "flops": flops}
    item = 2 if case["dtype"] == "bf16" else 4
    train = kind != "logprob" or case["train"]
    tokens = {"logprob": 8 + 4 + (4 if train else 0), "preference": 8 + 4, "policy": 8 + 8 + (4 if case.get("reference") else 0)}[kind]
    return {"bytes": counted * vocab * item + (rows * cols * item if train else 0) + rows * tokens,
            "flops": counted * vocab * (7 if train else 4)}

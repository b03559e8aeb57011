"""The post-training losses and gradient clipping through the pipeline engine on one GPU, against the fp32 oracle model."""
import importlib.util
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from oracle import gpt_ref  # noqa: E402

pytestmark = pytest.mark.gpu
CFG = gpt_ref.RefConfig(layers=2, hidden=128, heads=2, ffn=256, seq=64, vocab=500)
MB, GAS = 4, 3


def build(loss_fn, clipping=0.0, lr=1e-3):
    from bamboo_b200 import api, models
    from bamboo_b200.module import PipelineModule
    os.environ["BAMBOO_QUIET"] = "1"
    tc = models.TransformerConfig(layers=CFG.layers, hidden=CFG.hidden, heads=CFG.heads, ffn=CFG.ffn, seq=CFG.seq, vocab=CFG.vocab)
    model = PipelineModule(models.transformer_layer_specs(tc, 0), num_stages=1, loss_fn=loss_fn, partition_method="uniform")
    engine, *_ = api.initialize(model=model, config={
        "train_micro_batch_size_per_gpu": MB, "gradient_accumulation_steps": GAS, "bf16": {"enabled": True}, "gradient_clipping": clipping,
        "optimizer": {"type": "Adam", "params": {"lr": lr}}})
    engine.capture_grads = True
    return engine


def oracle_logps(P, tokens, targets):
    x = P["wte"][tokens] + P["wpe"][: tokens.shape[1]]
    for i in range(CFG.layers):
        x = gpt_ref.block_forward(CFG, P, f"b{i}.", x)
    x = torch.nn.functional.layer_norm(x, (CFG.hidden,), P["lnf_w"], P["lnf_b"], 1e-5)
    table = torch.log_softmax(torch.nn.functional.linear(x, P["head_w"]), -1)
    return table.gather(-1, targets.clamp(min=0)[..., None])[..., 0]


def oracle_gradient(loss_of, batches):
    P = {k: v.requires_grad_(True) for k, v in gpt_ref.init_params(CFG, 0).items()}
    losses = []
    for tokens, labels in batches:
        loss = loss_of(oracle_logps(P, tokens, labels[0]), *labels) / GAS
        loss.backward()
        losses.append(float(loss.detach()))
    return sum(losses), P


def synthetic(seed):
    g = torch.Generator().manual_seed(seed)
    P = gpt_ref.init_params(CFG, 0)
    out = []
    for _ in range(GAS):
        tokens = torch.randint(0, CFG.vocab, (MB, CFG.seq), generator=g)
        targets = torch.full_like(tokens, -100)
        targets[:, 8:-1] = tokens[:, 9:]
        with torch.no_grad():
            lp = oracle_logps(P, tokens, targets)
        # further from the clipping bounds than the bf16 model is from the fp32 one
        old = lp - torch.where(torch.rand(lp.shape, generator=g) < 0.5, 0.5, 0.02)
        out.append((tokens, targets, lp + 0.3 * torch.randn(lp.shape, generator=g), old, torch.randn(MB, generator=g)))
    return out


def preference(lp, targets, ref):
    s = torch.where(targets != -100, lp - ref, torch.zeros_like(lp)).sum(1)
    return torch.nn.functional.softplus(-0.1 * (s[0::2] - s[1::2])).mean()


def policy(lp, targets, old, adv, ref):
    keep = targets != -100
    ratio = (lp - old).exp()
    gap = ref - lp
    each = -torch.minimum(ratio * adv[:, None], ratio.clamp(0.8, 1.2) * adv[:, None]) + 0.1 * (gap.exp() - gap - 1)
    return each[keep].mean()


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_losses_through_the_engine_match_the_oracle(kind):
    from bamboo_b200 import lib, post_training as pt
    data = synthetic(3)
    if kind == "preference":
        loss_fn, loss_of = pt.PreferenceLoss(CFG.vocab, beta=0.1), preference
        batches = [(tokens, (targets, ref)) for tokens, targets, ref, _, _ in data]
    else:
        loss_fn, loss_of = pt.PolicyLoss(CFG.vocab, kl_coef=0.1), policy
        batches = [(tokens, (targets, old, adv, ref)) for tokens, targets, ref, old, adv in data]
    want, P = oracle_gradient(loss_of, batches)
    engine = build(loss_fn)
    got = float(engine.train_batch(data_iter=iter(batches)))
    # a bf16 model against an fp32 one: 2e-2 of the loss, 3e-2 of the gradient as a whole
    assert abs(got - want) <= 2e-2 * abs(want) + 2e-3
    names = ["wte", "wpe"] + [f"b{i}.{n}" for i in range(CFG.layers) for n in
                              ("ln1_w", "ln1_b", "qkv_w", "qkv_b", "proj_w", "proj_b", "ln2_w", "ln2_b", "fc1_w", "fc1_b", "fc2_w", "fc2_b")]
    names += ["lnf_w", "lnf_b", "head_w"]
    arena, flat = engine.arenas[0], engine.last_grads[0].cpu()
    ours = torch.cat([flat[off:off + n].view(arena.params[i].shape)[: P[name].shape[0]].reshape(-1)
                      for (i, off, n), name in zip(arena.named_slices(), names)])
    theirs = torch.cat([P[name].grad.reshape(-1) for name in names])
    assert ((ours - theirs).norm() / theirs.norm()).item() <= 3e-2
    assert lib.read_status() == 0


def test_clipping_inside_the_step_equals_clipping_before_it():
    """One step with `gradient_clipping` against a free engine's gradients, clipped in 64 bits and put through the Adam formula."""
    from bamboo_b200 import models, post_training as pt  # noqa: F401
    from bamboo_b200.layers import CrossEntropyLoss
    (batches,) = gpt_ref.synthetic_batches(CFG, MB, GAS, 1, seed=5)
    free, tight = build(CrossEntropyLoss(CFG.vocab)), build(CrossEntropyLoss(CFG.vocab), clipping=0.1)
    start = tight.arenas[0].master.clone()
    free.train_batch(data_iter=iter(batches))
    tight.train_batch(data_iter=iter(batches))
    assert free.get_global_grad_norm() is None
    g = tight.last_grads[0].double()
    norm = g.norm().item()
    assert norm > 0.1 and tight.get_global_grad_norm() == pytest.approx(norm, rel=1e-6)
    p = torch.nn.Parameter(start.double())
    p.grad = g * (0.1 / (norm + 1e-6))
    torch.optim.AdamW([p], lr=1e-3, weight_decay=0.0).step()
    moved = (p.detach() - start.double()).abs().max().item()
    assert ((tight.arenas[0].master.double() - p.detach()).abs().max().item()) <= 1e-4 * moved + 1e-8
    assert torch.equal(tight.arenas[0].lp, tight.arenas[0].master.bfloat16()) and torch.all(tight.arenas[0].grad == 0)


def test_the_example_learns():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "preference_tuning.py")
    spec = importlib.util.spec_from_file_location("preference_tuning", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    margins, gains = module.main(["--steps", "6"], log=lambda line: print(line))
    assert abs(margins[0]) < 1e-2 < margins[-1]            # policy = reference at first, then the preferred answers gain
    assert all(g > 0 for g in gains)

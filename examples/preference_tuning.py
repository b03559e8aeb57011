"""Post-training of a small GPT decoder on one GPU: preference pairs first, then a clipped policy loss, both through the pipeline engine.

    python examples/preference_tuning.py [--steps 8]

The task is synthetic: answers made of even token ids are preferred to answers of odd ones, and rewarded.  What a step runs:

* the reference model (the start weights) scores the tokens with ``head_logprobs``: hidden states, then the vocabulary projection
  without storing its logits;
* ``PreferenceLoss`` / ``PolicyLoss`` is the ``loss_fn`` of the policy's ``PipelineModule``; labels are a tuple of tensors;
* ``gradient_clipping`` in the configuration clips the global gradient norm inside the optimizer step.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from bamboo_b200 import models, post_training as pt  # noqa: E402
from bamboo_b200.api import initialize  # noqa: E402
from bamboo_b200.arena import ParamArena  # noqa: E402
from bamboo_b200.module import PipelineModule  # noqa: E402

CFG = models.GPT_TOY
MICRO_BATCH, MICRO_BATCHES, PROMPT = 4, 2, 32
IGNORE = -100


class Reference:
    """The frozen start weights: everything up to the vocabulary projection, and the projection's weight."""

    def __init__(self, specs):
        self.trunk = PipelineModule(specs[:-1], num_stages=1, loss_fn=None, partition_method="uniform")
        self.arena = ParamArena(self.trunk.stage_parameters(0), self.trunk.device, with_optimizer_state=False)
        self.head = specs[-1].build().weight.detach().to(self.trunk.device, torch.bfloat16)

    @torch.no_grad()
    def logprobs(self, tokens, targets):
        return pt.head_logprobs(self.trunk(tokens, stage_id=0), self.head, targets, CFG.vocab)


def policy_engine(specs, loss_fn):
    model = PipelineModule(specs, num_stages=1, loss_fn=loss_fn, partition_method="uniform")
    engine, *_ = initialize(model=model, config={
        "train_micro_batch_size_per_gpu": MICRO_BATCH, "gradient_accumulation_steps": MICRO_BATCHES, "bf16": {"enabled": True},
        "gradient_clipping": 1.0, "optimizer": {"type": "Adam", "params": {"lr": 2e-4}}})
    return engine


def answers(gen, parity):
    """Sequences of random tokens behind random prompts, the answers of sequence i all of parity[i]; (tokens, targets): a
    position's target is the next token, prompts and the last position do not count."""
    tokens = torch.randint(0, CFG.vocab, (MICRO_BATCH, CFG.seq), generator=gen)
    tokens[:, PROMPT:] = tokens[:, PROMPT:] // 2 * 2 + parity[:, None]
    targets = torch.full_like(tokens, IGNORE)
    targets[:, PROMPT - 1:-1] = tokens[:, PROMPT:]
    return tokens.cuda(), targets.cuda()


def preference_phase(specs, reference, steps, gen, log):
    """Sequence 2i (even answers) is preferred to 2i + 1 (odd ones)."""
    loss_fn = pt.PreferenceLoss(CFG.vocab, beta=0.1)
    engine = policy_engine(specs, loss_fn)
    margins = []
    for step in range(steps):
        batches = []
        for _ in range(MICRO_BATCHES):
            tokens, targets = answers(gen, torch.tensor([0, 1] * (MICRO_BATCH // 2)))
            batches.append((tokens, (targets, reference.logprobs(tokens, targets))))
        loss = float(engine.train_batch(data_iter=iter(batches)))
        margins.append(float((loss_fn.rewards[0::2] - loss_fn.rewards[1::2]).mean()))
        log(f"preference step {step}: loss {loss:.4f}, reward margin {margins[-1]:+.4f}, gradient norm {engine.get_global_grad_norm():.3f}")
    return margins


def policy_phase(specs, reference, steps, gen, log):
    """Answers of either parity, as if sampled; even ones have an advantage, odd ones the opposite."""
    loss_fn = pt.PolicyLoss(CFG.vocab, clip_low=0.2, clip_high=0.2, kl_coef=0.02)
    engine = policy_engine(specs, loss_fn)
    gains = []
    for step in range(steps):
        batches, before = [], []
        for _ in range(MICRO_BATCHES):
            parity = torch.randint(0, 2, (MICRO_BATCH,), generator=gen)
            tokens, targets = answers(gen, parity)
            advantages = (1.0 - 2.0 * parity).cuda()
            with torch.no_grad():       # the sampling policy's log-probabilities
                old = pt.token_logprobs(engine.module(tokens, stage_id=0), targets, CFG.vocab)
            batches.append((tokens, (targets, old, advantages, reference.logprobs(tokens, targets))))
            before.append((tokens, targets, advantages, old))
        loss = float(engine.train_batch(data_iter=iter(batches)))
        with torch.no_grad():
            gain = sum(((pt.token_logprobs(engine.module(t, stage_id=0), y, CFG.vocab) - old) * a[:, None]).sum() / (y != IGNORE).sum()
                       for t, y, a, old in before) / len(before)
        gains.append(float(gain))
        kl, clipped = loss_fn.stats.tolist()
        log(f"policy step {step}: loss {loss:+.4f}, gain {gains[-1]:+.5f}, KL {kl:.5f}, clipped {clipped:.3f}, "
            f"gradient norm {engine.get_global_grad_norm():.3f}")
    return gains


def main(argv=None, log=print):
    args = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    args.add_argument("--steps", type=int, default=8)
    args = args.parse_args(argv)
    os.environ.setdefault("BAMBOO_QUIET", "1")
    gen = torch.Generator().manual_seed(0)
    reference = Reference(models.transformer_layer_specs(CFG, seed=0))
    margins = preference_phase(models.transformer_layer_specs(CFG, seed=0), reference, args.steps, gen, log)
    gains = policy_phase(models.transformer_layer_specs(CFG, seed=0), reference, args.steps, gen, log)
    return margins, gains


if __name__ == "__main__":
    main()

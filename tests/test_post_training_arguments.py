"""What the post-training entry points make of their arguments, as far as that needs no GPU: the kernels are replaced by what records a call."""
import ctypes

import pytest
import torch


@pytest.fixture
def recorded(monkeypatch):
    """post_training with CPU tensors let through, and the descriptors that reach the native calls."""
    from bamboo_b200 import lib, post_training as pt
    seen = []

    def record(desc, *args, **kw):
        seen.append({name: getattr(desc, name) for name, _ in desc._fields_})
    for name in ("preference_loss", "policy_loss", "preference_loss_logits", "policy_loss_logits", "head_logprob_fwd"):
        monkeypatch.setattr(lib, name, record)
    monkeypatch.setattr(pt, "_on_current", lambda t, name: None)
    return pt, seen


def test_constants_given_as_tensors_are_read_at_every_call(recorded):
    pt, seen = recorded
    lp, t = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int64)
    x, h = torch.zeros(2, 4, 8), torch.zeros(8, 8, dtype=torch.bfloat16)
    value = torch.tensor(0.25)
    policy, preference = pt.PolicyLoss(8, kl_coef=value), pt.PreferenceLoss(8, beta=value)
    for want in (0.25, 0.5, 0.125):
        value.fill_(want)
        seen.clear()
        pt.policy_loss(lp, None, lp, t, kl_coef=value, clip_low=value, clip_high=value)
        pt.preference_loss(lp, None, t, beta=value, label_smoothing=value)
        policy.loss_and_grad(x, (t, None, lp))
        preference.loss_and_grad(x, t)
        pt.head_logprobs(h, h, t, temperature=value)
        assert [seen[0][n] for n in ("kl_coef", "clip_low", "clip_high")] == [want] * 3
        assert [seen[1][n] for n in ("beta", "label_smoothing")] == [want] * 2
        assert (seen[2]["kl_coef"], seen[3]["beta"], seen[4]["scale"]) == (want, want, 1 / want)

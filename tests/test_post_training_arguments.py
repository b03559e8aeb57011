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


def test_which_tensor_is_clipped(recorded):
    """A parameter of any class stands for its gradient, as in torch; a gradient for itself, one with a graph of its own included."""
    pt, _ = recorded
    parameter, leaf, arena, bare = torch.nn.Parameter(torch.ones(4)), torch.ones(4, requires_grad=True), torch.nn.Parameter(torch.ones(4)), torch.ones(4)
    parameter.grad, leaf.grad, arena.main_grad = torch.full((4,), 2.0), torch.full((4,), 3.0), torch.full((4,), 4.0)
    without = torch.ones(4, requires_grad=True)
    made = torch.ones(4, requires_grad=True) * 5
    assert not made.is_leaf
    grads = pt._gradients([parameter, leaf, arena, bare, without, made])[0]
    assert [g.data_ptr() for g in grads] == [t.data_ptr() for t in (parameter.grad, leaf.grad, arena.main_grad, bare, made)]
    assert [g.data_ptr() for g in pt._gradients(leaf)[0]] == [leaf.grad.data_ptr()]
    assert pt._gradients([without])[0] == []


def test_the_facade_clips_what_parameters_have_as_gradient(recorded, monkeypatch):
    import deepspeed.runtime.utils as ds_utils
    pt, _ = recorded
    seen = []
    monkeypatch.setattr(pt, "clip_grad_norm_", lambda tensors, max_norm: seen.append(list(tensors)) or torch.zeros(()))
    leaf, frozen, buffer = torch.ones(4, requires_grad=True), torch.nn.Parameter(torch.ones(4), requires_grad=False), torch.ones(4)
    leaf.grad = torch.full((4,), 3.0)
    arena = torch.nn.Parameter(torch.ones(4))
    arena.main_grad = torch.full((4,), 4.0)
    for given in ([leaf, frozen, buffer, arena], (p for p in (leaf, frozen, buffer, arena))):
        seen.clear()
        assert ds_utils.clip_grad_norm_(given, 1.0) == 0.0
        assert [t.data_ptr() for t in seen[0]] == [leaf.grad.data_ptr(), arena.main_grad.data_ptr()]
    ds_utils.clip_grad_norm_(leaf, 1.0)
    assert [t.data_ptr() for t in seen[1]] == [leaf.grad.data_ptr()]


def test_backward_pass_of_the_projection_refuses_rows_that_are_no_whole_vectors():
    """d_hidden, its fp32 parts and the copy of the hidden states have rows of ``hidden`` values, which are stored 16 bytes at a time."""
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20
    for hidden, weight_only in ((60, False), (12, False), (60, True), (1, False)):
        desc = lib.HeadDesc(rows=4, vocab=100, hidden=hidden, ld_hidden=64, ld_weight=64, scale=1.0, ignore_index=-100)
        rc = handle.bb_head_logprob_bwd(ctypes.byref(desc), at, at, at, at, at, None if weight_only else at, at, at, None, at, 104, at, 104, None)
        assert rc == -1 and b"bb_head_logprob_bwd" in handle.bb_last_error(), (hidden, rc, handle.bb_last_error())


def test_advantages_of_the_wrong_number_say_what_is_expected(recorded):
    pt, seen = recorded
    lp, t, offsets = torch.zeros(8), torch.zeros(8, dtype=torch.int64), torch.tensor([0, 3, 8])
    for call in (lambda a: pt.policy_loss(lp, None, a, t, offsets=offsets), lambda a: pt.PolicyLoss(4)(torch.zeros(8, 4), (t, None, a), offsets),
                 lambda a: pt.PolicyLoss(4).loss_and_grad(torch.zeros(8, 4), (t, None, a), offsets=offsets)):
        for count in (2, 5):
            with pytest.raises(ValueError, match=f"{count} values.*one per token.*repeat_interleave"):
                call(torch.zeros(count))
    with pytest.raises(ValueError, match="3 values.*8 tokens in 2 sequences"):
        pt.policy_loss(lp.view(2, 4), None, torch.zeros(3), t.view(2, 4))
    assert not seen
    pt.policy_loss(lp, None, torch.zeros(8), t, offsets=offsets)                                      # per token
    pt.policy_loss(lp.view(2, 4), None, torch.zeros(2), t.view(2, 4))                                 # per sequence, of one length
    assert [d["advantage_per_sequence"] for d in seen] == [0, 1]

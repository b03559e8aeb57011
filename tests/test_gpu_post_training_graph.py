"""The post-training functions inside an autograd graph: a graph that is kept for further backward passes, tensors that are overwritten,
second derivatives, attributes of a loss that change between forward and backward pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pt():
    from bamboo_b200 import lib, post_training
    lib.load()
    lib.read_status()
    return post_training


@pytest.fixture(autouse=True)
def healthy():
    yield
    from bamboo_b200 import lib
    torch.cuda.synchronize()
    assert lib.read_status() == 0


def batch(dtype=torch.float32, vocab=300):
    gen = torch.Generator(device="cuda").manual_seed(51)
    x = (torch.randn(4, 6, vocab, device="cuda", generator=gen) * 2).to(dtype)
    t = torch.randint(0, vocab, (4, 6), device="cuda", generator=gen)
    t[0, :2] = -100
    adv = torch.randn(4, 6, device="cuda", generator=gen)
    return x, t, adv


@pytest.mark.parametrize("vocab", [300, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss_over_a_kept_graph(pt, dtype, vocab):
    """Backward passes with other upstream gradients over one graph: each gets its own gradient, and those handed out before stay."""
    x, t, adv = batch(dtype, vocab)
    loss_fn = pt.PolicyLoss(vocab, inplace=False)
    _, _, unit = loss_fn.loss_and_grad(x, (t, None, adv), out=torch.empty_like(x))
    leaf = x.clone().requires_grad_(True)
    loss = loss_fn(leaf, (t, None, adv))
    handed = []
    for factor in (2.0, 2.0, 0.5, 0.0, 1.0):
        up = torch.tensor(factor, device="cuda")
        handed.append((factor, torch.autograd.grad(loss, leaf, up, retain_graph=True)[0]))
    for factor, grad in handed:
        assert torch.equal(grad, unit * factor)
    loss_fn.grad_scale = 0.25                                    # what a later call is to be made for
    for _ in range(2):
        assert torch.equal(torch.autograd.grad(loss, leaf, retain_graph=True)[0], unit)
    assert torch.equal(leaf.detach(), x)


def test_overwritten_logits_are_not_read_again(pt):
    """In place, the gradient stands where the logits were: a second backward pass is an error, as is one of an operation before that kept the
    logits themselves."""
    x, t, adv = batch()
    for call in (lambda y: pt.PolicyLoss(300)(y, (t, None, adv)), lambda y: pt.PreferenceLoss(300)(y, t),
                 lambda y: pt.token_logprobs(y, t, inplace=True).sum()):
        leaf = x.clone().requires_grad_(True)
        loss = call(leaf * 1.0)
        (first,) = torch.autograd.grad(loss, leaf, torch.tensor(0.5, device="cuda"), retain_graph=True)
        kept = first.clone()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, leaf, retain_graph=True)
        assert torch.equal(first, kept)
    leaf = x.clone().requires_grad_(True)
    loss = pt.PolicyLoss(300)(torch.tanh(leaf), (t, None, adv))                # (tanh keeps its output)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    want = torch.autograd.grad(pt.PolicyLoss(300, inplace=False)(torch.tanh(leaf), (t, None, adv)), leaf)[0]
    loss = pt.PolicyLoss(300)(torch.tanh(leaf) * 1.0, (t, None, adv))
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)


def test_graphs_that_are_not_overwritten_can_be_kept(pt):
    x, t, _ = batch()
    for call in (lambda y: pt.PreferenceLoss(300, inplace=False)(y, t), lambda y: pt.token_logprobs(y, t).sum()):
        leaf = x.clone().requires_grad_(True)
        loss = call(leaf)
        one = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], one)


def test_all_columns_are_the_vocabulary_where_none_is_given(pt):
    x, t, adv = batch()
    for make, labels in ((pt.PreferenceLoss, t), (pt.PolicyLoss, (t, None, adv))):
        grads = []
        for vocab in (300, None):
            leaf = x.clone().requires_grad_(True)
            make(vocab, inplace=False)(leaf, labels).backward()
            grads.append(leaf.grad)
        assert torch.equal(*grads)


def test_a_backward_pass_is_that_of_its_own_call(pt):
    """A loss whose vocabulary is changed for the next batch before the last one's backward pass."""
    x, t, adv = batch()
    t = t.clamp(max=199)
    for make, labels in ((pt.PreferenceLoss, t), (pt.PolicyLoss, (t, None, adv))):
        loss_fn = make(300, inplace=False)
        want = torch.autograd.grad(loss_fn(leaf := x.clone().requires_grad_(True), labels), leaf)[0]
        loss = loss_fn(leaf := x.clone().requires_grad_(True), labels)
        loss_fn.vocab, loss_fn.scale = 200, 2.0
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)


def test_second_derivatives_are_refused(pt):
    """They are not implemented, and a gradient that autograd took for a constant would be a wrong one."""
    x, t, adv = batch()
    h, w = torch.randn(24, 64, device="cuda").bfloat16(), torch.randn(300, 64, device="cuda").bfloat16()
    calls = ((lambda y: pt.token_logprobs(y, t).sum(), x), (lambda y: pt.PreferenceLoss(300, inplace=False)(y, t), x),
             (lambda y: pt.PolicyLoss(300, inplace=False)(y, (t, None, adv)), x), (lambda y: pt.head_logprobs(y, w, t.view(-1)).sum(), h),
             (lambda y: pt.preference_loss(y, None, t)[0], adv), (lambda y: pt.policy_loss(y, None, adv, t)[0], adv))
    for call, value in calls:
        leaf = value.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(call(leaf * 1.0) * 2.0, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grad.float().square().sum().backward()

"""The clipped policy loss where a ratio stands at a bound, and its KL term where policy and reference nearly agree."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
# a warp, 64, 128, 256 threads per row; rows in shared memory; rows too long for it
ROWS = [(4200, 500, F32), (4200, 4100, BF16), (4096, 5001, F32), (700, 16001, BF16), (1200, 50257, BF16), (300, 50257, F32), (150, 120001, BF16)]


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


@pytest.mark.parametrize("rows,vocab,dtype", ROWS)
def test_statistics_and_gradient_clip_the_same_tokens(pt, rows, vocab, dtype):
    """Ratios within a few steps of 32-bit numbers around a bound: the tokens without a gradient are those that the statistics count."""
    gen = torch.Generator(device="cuda").manual_seed(61)
    x = (torch.randn(rows, vocab, device="cuda", generator=gen) * 25).to(dtype)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    t = torch.where(t == x.argmax(1), (t + 1) % vocab, t)               # (a certain token has no gradient either)
    lp = torch.log_softmax(x.double(), 1).gather(1, t[:, None])[:, 0]
    up = torch.rand(rows, device="cuda", generator=gen) < 0.5
    old = (lp - torch.where(up, math.log(1.2), math.log(0.8))).float()
    steps = torch.randint(-2, 3, (rows,), device="cuda", generator=gen)
    for _ in range(2):
        old = torch.where(steps > 0, torch.nextafter(old, torch.full_like(old, 1e9)), torch.where(steps < 0, torch.nextafter(old, torch.full_like(old, -1e9)), old))
        steps = steps - steps.sign()
    adv = torch.where(up, 1.0, -1.0)
    _, stats, grad = pt.PolicyLoss(vocab).loss_and_grad(x, (t.view(1, -1), old, adv))
    without = (grad.gather(1, t[:, None])[:, 0] == 0).sum().item()
    assert 0 < without < rows
    assert stats[1].item() == pytest.approx(without / rows, rel=1e-6)


@pytest.mark.parametrize("rows,vocab,dtype", ROWS)
def test_slopes_of_improbable_tokens(pt, rows, vocab, dtype):
    """Log-probabilities of about -150: the ratio is a difference of two such numbers, and its error is that of the sum (2e-6), not of their
    rounding to 32 bits (1e-5)."""
    gen = torch.Generator(device="cuda").manual_seed(62)
    x = (torch.randn(rows, vocab, device="cuda", generator=gen) * 40).to(dtype)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    t = torch.where(t == x.argmax(1), (t + 1) % vocab, t)               # (a certain token has no gradient either)
    lp = torch.log_softmax(x.double(), 1).gather(1, t[:, None])[:, 0]
    old = (lp + 0.05).float()
    adv = torch.ones(rows, device="cuda")
    _, _, grad = pt.PolicyLoss(vocab).loss_and_grad(x.float(), (t.view(1, -1), old, adv))
    row = -(lp - old.double()).exp() / rows
    got = grad.double().gather(1, t[:, None])[:, 0]
    err = (got - row * -torch.expm1(lp)).abs()
    assert (err <= 4e-6 / rows).all(), err.max().item() * rows


@pytest.mark.parametrize("gap", [1e-4, 1e-3, 0.01, 0.1, 0.24, 0.26, 1.0, 3.0, -1e-4, -0.01, -0.24, -0.26, -1.0])
def test_kl_of_a_policy_near_its_reference(pt, gap):
    """e^gap - gap - 1 to 3e-6 of itself, from the gap between the 32-bit inputs (series below a quarter, the difference above)."""
    gen = torch.Generator(device="cuda").manual_seed(63)
    lp = -torch.rand(8, 40, device="cuda", generator=gen) * 3 - 1
    ref = lp + gap
    t = torch.zeros(8, 40, dtype=torch.int64, device="cuda")
    _, stats = pt.policy_loss(lp, None, torch.zeros(8, 40, device="cuda"), t, ref_logps=ref, kl_coef=1.0)
    g = ref.double() - lp.double()
    assert stats[0].item() == pytest.approx((torch.expm1(g) - g).mean().item(), rel=3e-6)


@pytest.mark.parametrize("mask", ["-inf", "lowest", "-1e30", "-1e5"])
@pytest.mark.parametrize("rows,vocab,dtype", ROWS)
def test_tokens_that_the_policy_rules_out(pt, rows, vocab, dtype, mask):
    """Targets that are masked: a ratio of 0, the clipped surrogate where the advantage is negative, and no gradient."""
    gen = torch.Generator(device="cuda").manual_seed(64)
    x = (torch.randn(rows, vocab, device="cuda", generator=gen) * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    masked = torch.rand(rows, device="cuda", generator=gen) < 0.5
    masked[:2] = torch.tensor([True, False])
    value = {"-inf": -math.inf, "lowest": torch.finfo(dtype).min}.get(mask) or float(mask)
    x[masked, t[masked]] = value
    lp, probs = torch.log_softmax(x.double(), 1).gather(1, t[:, None])[:, 0], torch.softmax(x.double(), 1)
    old = torch.where(masked, torch.full_like(lp, -5.0), lp + 0.1).float()
    adv = torch.randn(rows, device="cuda", generator=gen)
    ratio, a = (lp - old.double()).exp(), adv.double()
    want = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    loss, stats, grad = pt.PolicyLoss(vocab).loss_and_grad(x, (t.view(1, -1), old, adv))
    assert loss.item() == pytest.approx(want.mean().item(), rel=1e-5, abs=1e-6)
    assert stats[1].item() == pytest.approx((masked & (adv < 0)).sum().item() / rows, rel=1e-6)
    row = torch.where(masked, torch.zeros_like(a), -ratio * a / rows)[:, None]
    d = -row * probs
    d[torch.arange(rows, device="cuda"), t] += row[:, 0]
    err = (grad.double() - d).abs()
    assert (err <= (1.2e-5 if dtype == F32 else 2 ** -8) * d.abs() + 1e-6 * row.abs().max()).all()
    assert torch.all(grad[masked] == 0)

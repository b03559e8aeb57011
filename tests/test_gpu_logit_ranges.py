"""The row sums where the logits are far from a bell around zero: a low head of the vocabulary, low temperatures, large finite masks, against
the definitions in 64 bits, for every number of threads that a row is given, the cluster per row and the ring.

Tolerances.  A sum's reference may lie 2^64 below its terms, so arguments reach 64 in front of ex2: two roundings of 2^-19 each, 2.7e-6 of a
term after the factor ln 2, and ex2 and the sum as elsewhere (1e-6): log-probabilities 4e-6 + 1e-6 of their magnitude.  A gradient has
the same error once in its own exponential and once in the sum, and two roundings of arguments below 64 that its fewer parts of
the temperature bring: 1.2e-5 in fp32, 2^-8 in bf16, over 1e-7 of the largest incoming gradient."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


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


def near(got, want, rel, floor):
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    finite = torch.isfinite(want)
    assert torch.equal(got.double()[~finite], want[~finite])
    err = (got.double() - want).abs()
    bad = err[finite] > rel * want[finite].abs() + floor
    assert not bad.any(), (err[finite].max().item(), int(bad.sum()), rel, floor)


# (rows, vocabulary, type): a warp, 64, 128, 256 threads per row in each operator; 512 (gradients); a cluster per row; rows of the policy loss in
# shared memory by two CTAs and by one per SM, and too long for it
ROWS = [(4200, 2003, BF16), (4200, 1001, F32), (4200, 7000, BF16), (4100, 3000, F32), (4096, 16001, BF16), (1100, 30001, BF16), (1030, 9000, F32),
        (2100, 50257, BF16), (3, 50257, BF16), (2, 50257, F32), (40, 8192, F32), (700, 50257, F32), (160, 120001, BF16)]


def inputs(rows, vocab, dtype, pattern, seed):
    """Logits and temperature.  ``low``: the first part of the row, every thread's first chunk with it, 79 to 84 below the rest in
    steps that differ from row to row; ``flat``: the same over zeros; ``high``: the first part at 0 and 74 to 87 in the rest; ``cold``: a bell at
    a temperature of 0.05."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * 2
    head = min(vocab // 3, 4096)
    step = torch.linspace(0, 1, rows, device="cuda")[:, None]
    if pattern == "low":
        x[:, :head] = -79 - 5 * step
    elif pattern == "flat":
        x.zero_()
        x[:, :head] = -81 - 4 * step
    elif pattern == "high":
        x[:] = 74 + 13 * step
        x[:, :head] = 0
    return x.to(dtype), 0.05 if pattern == "cold" else 1.0, torch.randint(0, vocab, (rows,), device="cuda", generator=gen)


def reference(x, t, temperature):
    lp = torch.log_softmax(x.double() / temperature, 1)
    return lp.gather(1, t[:, None])[:, 0], lp.exp_()


@pytest.mark.parametrize("pattern", ["low", "flat", "high", "cold"])
@pytest.mark.parametrize("rows,vocab,dtype", ROWS)
def test_log_probabilities_and_gradients(pt, rows, vocab, dtype, pattern):
    x, temperature, t = inputs(rows, vocab, dtype, pattern, 31)
    lp, probs = reference(x, t, temperature)
    near(pt.token_logprobs(x, t, temperature=temperature), lp, 1e-6, 4e-6)
    g = torch.randn(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(32))
    leaf = x.requires_grad_(True)
    out = pt.token_logprobs(leaf, t, temperature=temperature)
    near(out.detach(), lp, 1e-6, 4e-6)
    out.backward(g)
    want = probs.mul_(-g.double()[:, None] / temperature)
    want[torch.arange(rows, device="cuda"), t] += g.double() / temperature
    near(leaf.grad, want, 1.2e-5 if dtype == F32 else 2 ** -8, 1e-7 * g.abs().max().item() / temperature)


@pytest.mark.parametrize("pattern", ["low", "flat", "high", "cold"])
@pytest.mark.parametrize("rows,vocab,dtype", ROWS)
def test_losses_and_their_gradients(pt, rows, vocab, dtype, pattern):
    """Both losses from logits.  The policy loss is computed from the log-probabilities in 64 bits: with log-probabilities of the sampling
    policy half below and half above them, each ratio away from the bounds of the clipping."""
    x, temperature, t = inputs(rows, vocab, dtype, pattern, 33)
    lp, probs = reference(x, t, temperature)
    gen = torch.Generator(device="cuda").manual_seed(34)
    old = (lp + torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.5, 0.1, -0.1)).float()
    adv = torch.randn(rows, device="cuda", generator=gen)
    ratio = (lp - old.double()).exp()
    loss, stats, grad = pt.PolicyLoss(vocab, temperature=temperature).loss_and_grad(x, (t.view(1, -1), old, adv))
    assert loss.item() == pytest.approx(-(ratio * adv.double()).mean().item(), rel=1e-5, abs=1e-5)
    assert stats[1].item() == 0
    row = (-ratio * adv.double() / rows / temperature)[:, None]
    want = -row * probs
    want[torch.arange(rows, device="cuda"), t] += row[:, 0]
    # (the ratio from a log-probability in 32 bits: its rounding, up to 3e-5 at 370, on top)
    near(grad, want, 5e-5 if dtype == F32 else 2 ** -8 + 5e-5, 1e-6 * row.abs().max().item())
    del want, grad
    even = rows // 2 * 2
    loss_fn = pt.PreferenceLoss(vocab, temperature=temperature, beta=0.05)
    loss, rewards, grad = loss_fn.loss_and_grad(x[:even], t[:even].view(even, 1))
    near(rewards, 0.05 * lp[:even], 1e-6, 1e-6)
    h = 0.05 * (lp[0:even:2] - lp[1:even:2])
    assert loss.item() == pytest.approx(torch.nn.functional.softplus(-h).mean().item(), rel=1e-5, abs=1e-6)
    slope = (torch.sigmoid(h) - 1) * 0.05 / (even // 2) / temperature
    row = torch.stack((slope, -slope), 1).reshape(-1, 1)
    want = -row * probs[:even]
    want[torch.arange(even, device="cuda"), t[:even]] += row[:, 0]
    near(grad, want, 1.5e-5 if dtype == F32 else 2 ** -8 + 2e-6, 1e-7 * row.abs().max().item())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_vocabularies_shorter_than_the_way_to_a_boundary(pt, dtype):
    """Rows that start anywhere, a vocabulary that ends before their first 16-byte boundary, and padding that goes on past it."""
    gen = torch.Generator(device="cuda").manual_seed(35)
    for vocab in range(1, 9):
        for cols in (vocab, vocab + 1, 9, 13, 17, 23, 40):
            if cols < vocab:
                continue
            rows = 19
            x = torch.randn(rows, cols, device="cuda", generator=gen).to(dtype)
            x[:, vocab:] = math.nan
            t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
            g = torch.randn(rows, device="cuda", generator=gen)
            lp, probs = reference(x[:, :vocab], t, 1.0)
            want = -g.double()[:, None] * probs
            want[torch.arange(rows, device="cuda"), t] += g.double()
            want = torch.nn.functional.pad(want, (0, cols - vocab))
            rel, floor = 1.2e-5 if dtype == F32 else 2 ** -8, 1e-7 * g.abs().max().item()
            for inplace in (False, True):
                leaf = x.clone().requires_grad_(True)
                out = pt.token_logprobs(leaf, t, vocab, inplace=inplace)
                near(out.detach(), lp, 1e-6, 4e-6)
                near(torch.autograd.grad(out, leaf, g)[0], want, rel, floor)
            y = x.clone()
            _, _, grad = pt.PolicyLoss(vocab).loss_and_grad(y, (t.view(1, -1), None, g), out=y)
            near(grad, -want / rows, rel, floor)
            y = x[:18].clone()
            _, _, grad = pt.PreferenceLoss(vocab, beta=1.0, form="hinge").loss_and_grad(y, t[:18].view(18, 1), out=y)
            h = lp[0:18:2] - lp[1:18:2]
            slope = torch.where(h < 1, -1.0, 0.0).double() / 9
            row = torch.stack((slope, -slope), 1).reshape(-1, 1)
            want = -row * probs[:18]
            want[torch.arange(18, device="cuda"), t[:18]] += row[:, 0]
            near(grad, torch.nn.functional.pad(want, (0, cols - vocab)), rel, 1e-7)


MASKS = [-1e5, -1e6, -1e9, -3e9, -1e10, -1e30, "half", "lowest"]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("rows,vocab,dtype", ROWS)
def test_large_finite_masks(pt, rows, vocab, dtype, mask):
    """Finite values that stand for "not this one", in parts of a row and in all of it, and their opposites.  Rows that lie whole
    beyond 2^20 in the exponent are summed over differences from their largest logit; below that the reference costs 2^-40 of the exponent."""
    lowest = torch.finfo(dtype).min
    value = {"half": lowest / 2, "lowest": lowest}.get(mask, mask)
    value = torch.tensor(value).to(dtype).item()
    temperature = 2.0 if MASKS.index(mask) % 2 else 1.0
    gen = torch.Generator(device="cuda").manual_seed(41)
    x = (torch.randn(rows, vocab, device="cuda", generator=gen) * 3).to(dtype)
    t = torch.randint(vocab // 2, vocab, (rows,), device="cuda", generator=gen)
    kind = torch.arange(rows, device="cuda") % 8
    if rows < 8:
        kind = (kind + MASKS.index(mask) * rows) % 8
    column = torch.arange(vocab, device="cuda")
    full = torch.full((), value, dtype=dtype, device="cuda")
    where = torch.where
    x = where((kind == 0)[:, None] & (column < vocab // 2), full, x)                   # the head
    x = where((kind == 1)[:, None] & (column != t[:, None]), full, x)                  # all but the target
    x = where((kind == 2)[:, None], full, x)                                           # all of it
    x = where((kind == 3)[:, None] & (column == t[:, None]), full, x)                  # the target
    x = where((kind == 4)[:, None] & (column // 64 % 2 == 0), full, x)                 # every other 64
    x = where((kind == 5)[:, None], torch.nextafter(full, -full) if dtype == F32 else full * 0.75, x)     # all, the target one step lower
    x = where((kind == 5)[:, None] & (column == t[:, None]), full, x)
    x = where((kind == 6)[:, None], -full, x)                                          # all of it, far above zero
    x = where((kind == 7)[:, None] & (column == t[:, None]), -full, x)                 # certain
    lp, probs = reference(x, t, temperature)
    near(pt.token_logprobs(x, t, temperature=temperature), lp, 1e-6, 4e-6)
    g = torch.randn(rows, device="cuda", generator=gen)
    leaf = x.requires_grad_(True)
    pt.token_logprobs(leaf, t, temperature=temperature).backward(g)
    want = probs.mul_(-g.double()[:, None] / temperature)
    want[torch.arange(rows, device="cuda"), t] += g.double() / temperature
    near(leaf.grad, want, 1.2e-5 if dtype == F32 else 2 ** -8, 1e-6 * g.abs().max().item() / temperature)
    loss, _, grad = pt.PolicyLoss(vocab, temperature=temperature).loss_and_grad(leaf.detach(), (t.view(1, -1), None, g))
    row = (-g.double() / rows / temperature)[:, None]
    near(grad, want * (row / (g.double()[:, None] / temperature)), 1.2e-5 if dtype == F32 else 2 ** -8, 1e-6 * row.abs().max().item())
    assert loss.item() == pytest.approx(-g.double().mean().item(), rel=1e-5, abs=1e-6)


def test_projected_logits_beyond_the_range_count_as_infinite(pt):
    """What a vocabulary projection's logits are from 2^31 in the exponent on: infinities of their sign, as the header states."""
    h = torch.zeros(3, 64, device="cuda", dtype=BF16)
    w = torch.zeros(300, 64, device="cuda", dtype=BF16)
    w[:, 0], w[:, 1], w[7, 1], w[:, 2] = 1e6, 1e6, -1e6, torch.linspace(-1, 1, 300, device="cuda").to(BF16)
    h[0, 0], h[1, 1], h[2, 2] = -1e6, -1e6, 1.0                  # all at -1e12; one at 1e12, the rest at -1e12; ordinary ones
    t = torch.tensor([5, 7, 9], device="cuda")
    hl = h.clone().requires_grad_(True)
    got = pt.head_logprobs(hl, w, t)
    assert got[0].item() == -math.inf and math.isnan(got[1].item())
    near(got[2:].detach(), reference(h[2:].double() @ w.double().t(), t[2:], 1.0)[0], 1e-6, 2e-5)
    got[0].backward()
    assert torch.all(hl.grad[0] == 0)

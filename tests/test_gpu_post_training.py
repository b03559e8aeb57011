"""The operators of a post-training step against their definitions in 64 bits, at the sizes, strides and masks where they can go
wrong, gradients against differences too, and what they refuse.

Tolerances follow from the arithmetic.  A log-probability is one rounding to fp32 (2^-24 relative) of a 64-bit value whose error
is that of a sum of up to 51200 ex2 results (2^-22 each, in the mean far less): 1e-6 of its magnitude plus 1e-6.  Gradients
are a softmax times the incoming gradient: relative 4e-6 in fp32 (two roundings of arguments below 64, one ex2, two products),
2^-8 in bf16 (half a unit in the last place and the fp32 error under it), absolute 1e-7 of the largest incoming gradient under
both.  Losses and rewards are sums of log-probabilities: their errors add up, at most tokens x 1e-6 x the size of one."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
IGNORE = -100


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


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def near(got, want, rel, floor):
    err = (got.double() - want).abs()
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    finite = torch.isfinite(want)
    assert torch.equal(got.double()[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
    bad = err[finite] > rel * want[finite].abs() + floor
    assert not bad.any(), (err[finite].max().item(), rel, floor)


def logits_of(rows, vocab, cols, dtype, seed, spread=3.0):
    x = torch.randn(rows, cols, device="cuda", generator=gen(seed)) * spread
    return x.to(dtype)


def targets_of(rows, vocab, seed, ignored=0.2):
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(seed + 1))
    t[torch.rand(rows, device="cuda", generator=gen(seed + 2)) < ignored] = IGNORE
    return t


def ref_logps(logits, targets, vocab, temperature=1.0):
    """64-bit log-probabilities and softmax; a row without any finite logit has neither: -inf, zeros."""
    x = logits[:, :vocab].double() / temperature
    counted = targets != IGNORE
    logp = torch.log_softmax(x, 1)
    empty = (x == -math.inf).all(1)
    lp = logp.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
    return torch.where(counted, lp, torch.zeros_like(lp)), torch.where(empty[:, None], torch.zeros_like(logp), logp.exp()), counted & ~empty


def ref_dlogits(probs, counted, targets, row_grad, cols, temperature=1.0):
    g = torch.where(counted, row_grad.double(), torch.zeros((), dtype=torch.float64, device="cuda")) / temperature
    d = -g[:, None] * probs
    d = torch.where(counted[:, None], d, torch.zeros_like(d))
    d[torch.arange(len(g), device="cuda"), targets.clamp(min=0)] += g
    return torch.nn.functional.pad(d, (0, cols - probs.shape[1]))


# ----------------------------------------------------------------------------------- token log-probabilities
SHAPES = [(1, 1, 1), (5, 1, 8), (3, 7, 7), (4, 1000, 1024), (1, 50257, 50257), (9, 50257, 50304), (150, 257, 257), (700, 333, 336),
          (2, 51200, 51200), (65, 8192, 8200), (300, 2049, 2049), (1, 200003, 200003), (600, 4096, 4097)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,cols", SHAPES)
def test_token_logprobs_and_gradient(pt, rows, vocab, cols, dtype):
    x, t = logits_of(rows, vocab, cols, dtype, 3), targets_of(rows, vocab, 4)
    g = torch.randn(rows, device="cuda", generator=gen(5))
    for temperature in (1.0, 0.7):
        lp, probs, counted = ref_logps(x, t, vocab, temperature)
        got = pt.token_logprobs(x, t, vocab, temperature=temperature)
        near(got, lp, 1e-6, 1e-6)
        leaf = x.clone().requires_grad_(True)
        out = pt.token_logprobs(leaf, t, vocab, temperature=temperature)
        near(out.detach(), lp, 1e-6, 1e-6)
        out.backward(g)
        want = ref_dlogits(probs, counted, t, g, cols, temperature)
        near(leaf.grad, want, 4e-6 if dtype == torch.float32 else 2 ** -8, 1e-7 * g.abs().max().item() / temperature)
        assert torch.all(leaf.grad[:, vocab:] == 0) and torch.all(leaf.grad[t == IGNORE] == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5])
def test_rows_that_start_anywhere(pt, dtype, offset):
    """A window of a wider matrix, at every alignment; the columns around it stay as they are."""
    rows, vocab, ld = 33, 1003, 1021
    whole = logits_of(rows, ld, ld, dtype, 7)
    x, t = whole[:, offset:offset + vocab], targets_of(rows, vocab, 8)
    lp, probs, counted = ref_logps(x, t, vocab)
    near(pt.token_logprobs(x, t), lp, 1e-6, 1e-6)
    g = torch.randn(rows, device="cuda", generator=gen(9))
    want = ref_dlogits(probs, counted, t, g, vocab)
    tol = 4e-6 if dtype == torch.float32 else 2 ** -8
    leaf = whole.clone().requires_grad_(True)
    pt.token_logprobs(leaf[:, offset:offset + vocab], t).backward(g)
    near(leaf.grad[:, offset:offset + vocab], want, tol, 1e-7 * g.abs().max().item())
    before = whole.clone()
    part = whole[:, offset:offset + vocab].detach().requires_grad_(True)      # the gradient over the logits
    (grad,) = torch.autograd.grad(pt.token_logprobs(part, t, inplace=True), part, g)
    near(grad, want, tol, 1e-7 * g.abs().max().item())
    assert grad.data_ptr() == part.data_ptr()
    assert torch.equal(whole[:, :offset], before[:, :offset]) and torch.equal(whole[:, offset + vocab:], before[:, offset + vocab:])


def test_other_strides_and_shapes(pt):
    x = logits_of(6 * 5, 77, 77, torch.float32, 11).view(6, 5, 77)
    t = targets_of(30, 77, 12).view(6, 5)
    want = ref_logps(x.reshape(30, 77), t.reshape(-1), 77)[0].view(6, 5)
    near(pt.token_logprobs(x, t), want, 1e-6, 1e-6)
    near(pt.token_logprobs(x.transpose(0, 1).contiguous().transpose(0, 1), t), want, 1e-6, 1e-6)       # rows in another order
    near(pt.token_logprobs(x.permute(2, 0, 1).contiguous().permute(1, 2, 0), t), want, 1e-6, 1e-6)     # vocabulary outermost
    near(pt.token_logprobs(x[:, 1:], t[:, 1:]), want[:, 1:], 1e-6, 1e-6)
    near(pt.token_logprobs(x[:1].expand(6, 5, 77), t[:1].expand(6, 5)), want[:1].expand(6, 5), 1e-6, 1e-6)
    assert pt.token_logprobs(x[:0], t[:0]).shape == (0, 5)
    near(pt.token_logprobs(x[:, 2:3], t[:, 2:3]), want[:, 2:3], 1e-6, 1e-6)                            # one token of each sequence
    near(pt.token_logprobs(x[:, 2], t[:, 2]), want[:, 2], 1e-6, 1e-6)
    near(pt.token_logprobs(x[3, 2], t[3, 2]).reshape(1), want[3, 2].reshape(1), 1e-6, 1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_vocabulary_and_values_in_ignored_rows(pt, dtype):
    """-inf and the type's lowest value as masks, a row without any logit left, NaN and infinities where nothing counts."""
    rows, vocab = 12, 1001
    x = logits_of(rows, vocab, vocab, dtype, 13)
    t = torch.arange(rows, device="cuda") * 7
    lowest = torch.finfo(dtype).min
    x[0, 100:] = -math.inf
    x[1, :500] = lowest
    t[1] = 600
    x[2] = -math.inf                      # no distribution
    x[3, 5:] = -math.inf
    t[3] = 900                            # the target itself is masked
    x[4, :] = -math.inf
    x[4, 17] = 1.0
    t[4] = 17                             # certain
    x[5], t[5] = math.nan, IGNORE
    x[6], t[6] = math.inf, IGNORE
    x[7] = lowest                         # a uniform row at the bottom of the range
    x[8, 3] = math.nan                    # NaN in a counted row stays visible
    x[9] = 80.0                           # a uniform row far from zero
    lp, probs, counted = ref_logps(x, t, vocab)
    near(pt.token_logprobs(x, t), lp, 1e-6, 1e-6)
    g = torch.ones(rows, device="cuda")
    leaf = x.clone().requires_grad_(True)
    pt.token_logprobs(leaf, t).backward(g)
    want = ref_dlogits(probs, counted, t, g, vocab)
    near(leaf.grad, want, 4e-6 if dtype == torch.float32 else 2 ** -8, 1e-7)
    assert torch.all(leaf.grad[[2, 5, 6]] == 0)


def test_gradient_of_log_probabilities_against_differences(pt):
    """Central differences of the 64-bit definition along random directions."""
    rows, vocab = 7, 301
    x, t = logits_of(rows, vocab, vocab, torch.float32, 15), targets_of(rows, vocab, 16, 0.0)
    g = torch.randn(rows, device="cuda", generator=gen(17)).double()
    leaf = x.clone().requires_grad_(True)
    pt.token_logprobs(leaf, t, temperature=1.3).backward(g.float())
    for seed in range(3):
        v = torch.randn(rows, vocab, device="cuda", generator=gen(18 + seed)).double()
        h = 1e-5
        f = lambda z: (g * torch.log_softmax(z / 1.3, 1).gather(1, t[:, None])[:, 0]).sum()  # noqa: E731
        slope = ((f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)).item()
        assert abs((leaf.grad.double() * v).sum().item() - slope) <= 1e-5 * (leaf.grad.double().norm() * v.norm()).item()


def test_targets_outside_the_vocabulary_are_reported(pt):
    from bamboo_b200 import lib
    x, t = logits_of(4, 100, 104, torch.bfloat16, 19), torch.tensor([1, 100, -1, 7], device="cuda")
    got = pt.token_logprobs(x, t, 100)
    torch.cuda.synchronize()
    assert lib.read_status() < 0
    assert got[1] == 0 and got[2] == 0 and got[0] != 0


# ----------------------------------------------------------------------------------- through the vocabulary projection
def ref_head(h, w, t, vocab, temperature, g=None):
    """64-bit log-probabilities and, for an incoming gradient, the gradients of hidden states and weight."""
    h, w = h.double(), w.double()
    lp, probs, counted = ref_logps(h @ w[:vocab].t(), t, vocab, temperature)
    if g is None:
        return lp
    d = ref_dlogits(probs, counted, t, g, w.shape[0], temperature)
    return lp, d @ w, d.t() @ h


# Logits are fp32 sums of up to 4096 bf16 products of size 1 / hidden: 1e-5 at most; log-probabilities 1e-6 of their magnitude on top.
# The logit gradient is rounded to bf16 (2^-8 of each), the results too; sums of such errors stay below 2^-7 of the sums of magnitudes.
HEAD_SHAPES = [(1, 64, 300, 300), (1, 1024, 50257, 50304), (3, 8, 1, 1), (128, 256, 1000, 1024), (129, 264, 257, 257), (300, 520, 2049, 2056),
               (1000, 128, 30522, 30592), (2500, 64, 5000, 5000), (7, 4096, 777, 777), (40, 72, 128, 128), (700, 1024, 12345, 12345)]


@pytest.mark.parametrize("rows,hidden,vocab,cols", HEAD_SHAPES)
def test_head_logprobs_and_gradients(pt, rows, hidden, vocab, cols):
    h = torch.randn(rows, hidden, device="cuda", generator=gen(101)).bfloat16()
    w = (torch.randn(cols, hidden, device="cuda", generator=gen(102)) * 2 / math.sqrt(hidden)).bfloat16()
    t = targets_of(rows, vocab, 103)
    g = torch.randn(rows, device="cuda", generator=gen(104))
    lp, dh, dw = ref_head(h, w, t, vocab, 0.8, g)
    near(pt.head_logprobs(h, w, t, vocab, temperature=0.8), lp, 1e-6, 2e-5)
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    pt.head_logprobs(hl, wl, t, vocab, temperature=0.8).backward(g)
    d = (ref_dlogits(*ref_logps(h.double() @ w[:vocab].double().t(), t, vocab, 0.8)[1:], t, g, cols, 0.8)).abs()
    for got, want, size in ((hl.grad, dh, d @ w.double().abs()), (wl.grad, dw, d.t() @ h.double().abs())):
        assert ((got.double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -7 * size + 1e-6).all()
    assert torch.all(wl.grad[vocab:] == 0) and torch.all(hl.grad[t == IGNORE] == 0)


def test_head_backward_in_pieces_and_into_an_arena(pt, monkeypatch):
    """Pieces of the vocabulary give the gradients of the whole, and a weight with ``main_grad`` is added to there."""
    rows, hidden, vocab, cols = 300, 128, 5003, 5120
    h = torch.randn(rows, hidden, device="cuda", generator=gen(105)).bfloat16()
    w = (torch.randn(cols, hidden, device="cuda", generator=gen(106)) * 0.2).bfloat16()
    t, g = targets_of(rows, vocab, 107), torch.randn(rows, device="cuda", generator=gen(108))
    whole = torch.autograd.grad(pt.head_logprobs(hl := h.clone().requires_grad_(True), wl := w.clone().requires_grad_(True), t, vocab), (hl, wl), g)
    monkeypatch.setattr(pt, "HEAD_GRAD_BYTES", 1)                   # the least: 2048 entries at a time
    pieces = torch.autograd.grad(pt.head_logprobs(hl, wl, t, vocab), (hl, wl), g)
    assert torch.equal(whole[1], pieces[1])
    near(pieces[0], whole[0].double(), 2 ** -7, 2 ** -8 * whole[0].abs().max().item())
    p = torch.nn.Parameter(w.clone())
    p.main_grad = torch.ones(cols, hidden, device="cuda")
    pt.head_logprobs(h, p, t, vocab).backward(g)
    assert p.grad is None
    near((p.main_grad - 1).bfloat16(), whole[1].double(), 2 ** -7, 1e-6)


@pytest.mark.parametrize("rows,hidden,vocab,parts", [(64, 768, 50257, True), (411, 792, 36348, True), (1999, 768, 32000, True), (130, 2304, 600, False)])
def test_head_gradient_in_parts_of_the_vocabulary(pt, rows, hidden, vocab, parts, monkeypatch):
    from bamboo_b200 import lib
    desc = lib.HeadDesc(rows=rows, vocab=vocab, hidden=hidden, ld_hidden=hidden, ld_weight=hidden, scale=1.0, ignore_index=IGNORE)
    assert (lib.head_bwd_parts(desc, (vocab + 7) // 8 * 8) > 1) == parts and lib.head_bwd_parts(desc, 256) >= 1
    h = torch.randn(rows, hidden, device="cuda", generator=gen(81)).bfloat16()
    w = (torch.randn(vocab, hidden, device="cuda", generator=gen(82)) / hidden ** 0.5).bfloat16()
    t, g = targets_of(rows, vocab, 83), torch.randn(rows, device="cuda", generator=gen(84))
    dh = ref_head(h, w, t, vocab, 1.0, g)[1]
    size = ref_dlogits(*ref_logps(h.double() @ w.double().t(), t, vocab)[1:], t, g, vocab).abs() @ w.double().abs()
    whole = None
    for limit in (256 << 20, 2 * rows * 4096):          # the vocabulary at once, and in pieces of 4096
        monkeypatch.setattr(pt, "HEAD_GRAD_BYTES", limit)
        for _ in range(3):
            leaf = h.clone().requires_grad_(True)
            pt.head_logprobs(leaf, w, t, vocab).backward(g)
            assert ((leaf.grad.double() - dh).abs() <= 2 ** -8 * dh.abs() + 2 ** -7 * size + 1e-6).all()
            assert whole is None or torch.equal(leaf.grad, whole)      # parts are added up in one order
            whole = leaf.grad
        whole = None


def test_head_operands_of_other_layouts(pt):
    h = torch.randn(4, 9, 96, device="cuda", generator=gen(109)).bfloat16()
    w = (torch.randn(400, 104, device="cuda", generator=gen(110)) * 0.2).bfloat16()
    t = targets_of(36, 333, 111).view(4, 9)
    for wv in (w[:, :96], w[:, 1:97], w[3:, 8:], w.t()[:96].t()):
        for hv in (h, h.transpose(0, 1).contiguous().transpose(0, 1), h[:, 1:]):
            tv = t[:, :hv.shape[1]]
            want = ref_head(hv.reshape(-1, 96), wv, tv.reshape(-1), 333, 1.0)
            near(pt.head_logprobs(hv, wv, tv, 333).reshape(-1), want, 1e-6, 2e-5)
    assert pt.head_logprobs(h[:0], w[:, :96], t[:0]).shape == (0, 9)


def test_head_gradient_against_differences(pt):
    rows, hidden, vocab = 6, 32, 211
    h = torch.randn(rows, hidden, device="cuda", generator=gen(112)).bfloat16()
    w = (torch.randn(vocab, hidden, device="cuda", generator=gen(113)) * 0.3).bfloat16()
    t, g = targets_of(rows, vocab, 114, 0.0), torch.randn(rows, device="cuda", generator=gen(115)).double()
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    pt.head_logprobs(hl, wl, t).backward(g.float())
    f = lambda a, b: (g * torch.log_softmax(a @ b.t(), 1).gather(1, t[:, None])[:, 0]).sum()  # noqa: E731
    for seed in range(3):
        v = torch.randn(rows, hidden, device="cuda", generator=gen(116 + seed)).double()
        u = torch.randn(vocab, hidden, device="cuda", generator=gen(126 + seed)).double()
        e = 1e-5
        slope_h = (f(h.double() + e * v, w.double()) - f(h.double() - e * v, w.double())) / (2 * e)
        slope_w = (f(h.double(), w.double() + e * u) - f(h.double(), w.double() - e * u)) / (2 * e)
        # bf16 roundings, independent of the direction
        assert abs((hl.grad.double() * v).sum() - slope_h) <= 2 ** -7 * hl.grad.double().norm() * v.norm()
        assert abs((wl.grad.double() * u).sum() - slope_w) <= 2 ** -7 * wl.grad.double().norm() * u.norm()


def test_head_rows_that_do_not_count_and_refusals(pt):
    from bamboo_b200 import lib
    h = torch.randn(5, 64, device="cuda", generator=gen(119)).bfloat16()
    w = (torch.randn(100, 64, device="cuda", generator=gen(120)) * 0.2).bfloat16()
    t = torch.tensor([3, IGNORE, 99, IGNORE, 0], device="cuda")
    want = ref_head(h, w, t, 100, 1.0)
    h[1], h[3] = math.nan, math.inf
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = pt.head_logprobs(hl, wl, t)
    near(out.detach(), want, 1e-6, 2e-5)
    out.sum().backward()
    assert torch.isfinite(hl.grad).all() and torch.all(hl.grad[[1, 3]] == 0)
    assert torch.isfinite(wl.grad).all()                  # zero times NaN of a row that does not count stays out of it
    p = torch.nn.Parameter(w.clone())
    p.main_grad = torch.zeros(100, 64, device="cuda")
    pt.head_logprobs(h, p, t).sum().backward()
    near(p.main_grad.bfloat16(), wl.grad.double(), 2 ** -7, 1e-6)
    out = pt.head_logprobs(h, w, torch.tensor([3, 100, -7, IGNORE, 0], device="cuda"))
    torch.cuda.synchronize()
    assert lib.read_status() < 0 and torch.all(out[1:4] == 0)
    with pytest.raises(ValueError):
        pt.head_logprobs(h, w, t, 101)
    with pytest.raises(ValueError):
        pt.head_logprobs(h[:, :60], w[:, :60], t)
    with pytest.raises(ValueError):
        pt.head_logprobs(h, w[:, :56], t)
    with pytest.raises(lib.BambooNativeError):
        pt.head_logprobs(h.float(), w, t)
    with pytest.raises(lib.BambooNativeError):
        pt.head_logprobs(h, w.cpu(), t)


# ----------------------------------------------------------------------------------- preference loss
def spans_of(lengths):
    ends = torch.tensor(lengths).cumsum(0).tolist()
    return list(zip([0] + ends[:-1], ends))


def ref_preference(lp, ref, counted, spans, beta, form, smoothing, average):
    scores = []
    for a, b in spans:
        keep = counted[a:b]
        s = (lp[a:b] - ref[a:b])[keep].sum()
        scores.append(s / max(1, int(keep.sum())) if average else s)
    s = torch.stack(scores)
    h = beta * (s[0::2] - s[1::2])
    if form == "sigmoid":
        each = -(1 - smoothing) * torch.nn.functional.logsigmoid(h) - smoothing * torch.nn.functional.logsigmoid(-h)
    elif form == "hinge":
        each = torch.relu(1 - h)
    else:
        each = (h / beta - 1 / (2 * beta)) ** 2
    return each.mean(), beta * s


LENGTHS = [[1, 1], [5, 0], [0, 0, 3, 4], [17, 300, 1, 64], [1000, 24, 513, 7, 0, 9], [64] * 8]


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("form,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("squared", 0.0)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_preference_loss_over_logprobs(pt, lengths, form, smoothing, average):
    n = sum(lengths)
    lp = -3 * torch.rand(n, device="cuda", generator=gen(21))
    ref = lp + 0.3 * torch.randn(n, device="cuda", generator=gen(22))
    t = targets_of(n, 50, 23, 0.3)
    if len(lengths) == 4:
        t[lengths[0]:lengths[0] + lengths[1]] = IGNORE       # a sequence that is all prompt
    lp[t == IGNORE], ref[t == IGNORE] = math.nan, math.inf
    offsets = torch.tensor([a for a, _ in spans_of(lengths)] + [n], device="cuda")
    leaf = lp.clone().requires_grad_(True)
    loss, rewards = pt.preference_loss(leaf, ref, t, beta=0.3, form=form, label_smoothing=smoothing, average=average, offsets=offsets)
    (3.0 * loss).backward()
    exact = lp.double().requires_grad_(True)
    want, want_rewards = ref_preference(exact, ref.double(), t != IGNORE, spans_of(lengths), 0.3, form, smoothing, average)
    (grad,) = torch.autograd.grad(3.0 * want, exact)
    # sums in 64 bits: what is left is the rounding of the results, and the product with the upstream gradient
    near(loss.detach().reshape(1), want.detach().reshape(1), 1e-6, 1e-7)
    near(rewards, want_rewards.detach(), 1e-6, 1e-7)
    near(leaf.grad, torch.nan_to_num(grad), 1e-6, 1e-9)
    if len(set(lengths)) == 1:
        again, _ = pt.preference_loss(lp.view(len(lengths), -1), ref.view(len(lengths), -1), t.view(len(lengths), -1), beta=0.3, form=form,
                                      label_smoothing=smoothing, average=average)
        assert again == loss


def test_preference_without_reference_and_at_extremes(pt):
    t = torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    lp = torch.tensor([[-1e4, -1e4, -1e4], [0.0, 0.0, 0.0], [0.0, 0.0, 0.0], [-1e4, -1e4, -1e4]], device="cuda").requires_grad_(True)
    loss, rewards = pt.preference_loss(lp, None, t, beta=1.0)
    loss.backward()
    near(loss.detach().reshape(1), torch.tensor([15000.0], dtype=torch.float64, device="cuda"), 1e-6, 0)
    near(rewards, torch.tensor([-3e4, 0, 0, -3e4], dtype=torch.float64, device="cuda"), 1e-6, 0)
    assert torch.equal(lp.grad[:2], torch.tensor([[-0.5] * 3, [0.5] * 3], device="cuda")) and torch.all(lp.grad[2:] == 0)


def test_many_pairs_are_summed_in_one_order(pt):
    pairs, length = 700, 31
    lp = -torch.rand(2 * pairs, length, device="cuda", generator=gen(25))
    ref = -torch.rand(2 * pairs, length, device="cuda", generator=gen(26))
    t = torch.zeros(2 * pairs, length, dtype=torch.int64, device="cuda")
    a, _ = pt.preference_loss(lp, ref, t)
    b, _ = pt.preference_loss(lp, ref, t)
    want, _ = ref_preference(lp.double().view(-1), ref.double().view(-1), (t == 0).view(-1), spans_of([length] * 2 * pairs), 0.1, "sigmoid", 0.0, False)
    assert torch.equal(a, b)
    near(a.reshape(1), want.reshape(1), 1e-6, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,cols,shape", [(1000, 1024, (4, 33)), (777, 777, (2, 1)), (50257, 50304, (2, 40)), (5000, 5001, (6, 50))])
def test_preference_loss_from_logits(pt, dtype, vocab, cols, shape):
    rows = shape[0] * shape[1]
    x, t = logits_of(rows, vocab, cols, dtype, 27), targets_of(rows, vocab, 28)
    lp, probs, counted = ref_logps(x, t, vocab, 0.9)
    ref = (lp + 0.2 * torch.randn(rows, device="cuda", generator=gen(29)).double()).float()
    exact = lp.clone().requires_grad_(True)
    want, want_rewards = ref_preference(exact, ref.double(), t != IGNORE, spans_of([shape[1]] * shape[0]), 0.1, "sigmoid", 0.1, False)
    (row_grad,) = torch.autograd.grad(want, exact)
    dx = ref_dlogits(probs, counted, t, row_grad, cols, 0.9)
    loss_fn = pt.PreferenceLoss(vocab, beta=0.1, label_smoothing=0.1, temperature=0.9, inplace=False)
    labels = (t.view(shape), ref.view(shape))
    # the slope of the loss carries the error of the rewards, themselves sums of shape[1] log-probabilities
    err = 0.1 * shape[1] * 1e-6 * (1 + lp.abs().max().item())
    tol = (4e-6 if dtype == torch.float32 else 2 ** -8) + 2 * err
    loss, rewards, grad = loss_fn.loss_and_grad(x.view(*shape, cols), labels, grad_scale=0.25)
    near(loss.reshape(1), want.detach().reshape(1), 1e-6, err)
    near(rewards, want_rewards.detach(), 1e-6, err)
    near(grad.view(rows, cols), 0.25 * dx, tol, 1e-7 * row_grad.abs().max().item())
    leaf = x.clone().requires_grad_(True)
    (loss_fn(leaf.view(*shape, cols), labels) * 0.25).backward()
    assert torch.equal(leaf.grad, grad.view(rows, cols))
    with torch.no_grad():
        assert loss_fn(x.view(*shape, cols), labels) == loss
    over = x.clone().view(*shape, cols)
    out = loss_fn.loss_and_grad(over, labels, out=over, grad_scale=0.25)[2]
    assert out is over and torch.equal(over.view(rows, cols), grad.view(rows, cols))


@pytest.mark.parametrize("vocab", [257, 32000])
def test_rewards_of_a_policy_that_is_its_reference(pt, vocab):
    # The reference's log-probabilities are the policy's own, rounded to fp32: the rewards are what that rounding left out.  A sum of
    # vocab ex2 results, 2^-22 at most each and of either sign, is some 2^-24 off; rounding the policy's values too would add 3e-7.
    rows = 512
    x, t = logits_of(rows, vocab, vocab, torch.float32, 37), targets_of(rows, vocab, 38, 0.0)
    lp, _, _ = ref_logps(x, t, vocab)
    loss, rewards, _ = pt.PreferenceLoss(vocab, beta=1.0, inplace=False).loss_and_grad(x.view(rows, 1, vocab), (t.view(rows, 1), lp.float().view(rows, 1)))
    off = rewards.double() - (lp - lp.float().double())
    assert off.square().mean().sqrt().item() <= 2 ** -23
    near(loss.reshape(1), torch.tensor([math.log(2)], dtype=torch.float64, device="cuda"), 1e-6, 0)


# ----------------------------------------------------------------------------------- policy loss
def ref_policy(lp, old, adv, ref, counted, spans, low, high, kl_coef, reduction):
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    ratio = torch.where(counted, lp - old, zero).exp() if old is not None else torch.where(counted, lp - lp.detach(), zero).exp()
    adv = torch.where(counted, adv, zero)
    plain, bounded = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    clipped = (bounded < plain) & counted
    each = -torch.where(clipped, bounded, plain)
    kl = torch.zeros_like(each)
    if ref is not None:
        gap = torch.where(counted, ref - lp, zero)
        kl = gap.exp() - gap - 1
        each = each + kl_coef * kl
    total = max(1, int(counted.sum()))
    if reduction == "token":
        loss = torch.where(counted, each, zero).sum() / total
    else:
        loss = sum((each[a:b][counted[a:b]].sum() / max(1, int(counted[a:b].sum())) for a, b in spans), zero) / len(spans)
    return loss, torch.stack([torch.where(counted, kl, zero).sum() / total, clipped.sum().double() / total])


def policy_inputs(lp, seed):
    """Old log-probabilities whose ratios keep clear of the bounds 0.8 and 1.3, advantages of both signs and one exact zero."""
    n = lp.numel()
    moved = 0.3 * torch.randn(n, device="cuda", generator=gen(seed)).double()
    for bound in (math.log(0.8), math.log(1.3)):
        moved = torch.where((moved - bound).abs() < 1e-3, moved + 4e-3, moved)
    adv = torch.randn(n, device="cuda", generator=gen(seed + 1))
    adv[n // 2] = 0
    return (lp - moved).float(), adv, (lp + 0.2 * torch.randn(n, device="cuda", generator=gen(seed + 2)).double()).float()


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("kl_coef,on_policy", [(0.0, False), (0.1, False), (0.1, True)])
@pytest.mark.parametrize("lengths", LENGTHS + [[40000, 3]], ids=str)
def test_policy_loss_over_logprobs(pt, lengths, kl_coef, on_policy, reduction):
    n = sum(lengths)
    lp = -3 * torch.rand(n, device="cuda", generator=gen(31))
    old, adv, ref = policy_inputs(lp.double(), 32)
    t = targets_of(n, 50, 35, 0.3)
    if len(lengths) == 4:
        t[lengths[0]:lengths[0] + lengths[1]] = IGNORE
    for v in (lp, old, adv, ref):
        v[t == IGNORE] = math.nan
    offsets = torch.tensor([a for a, _ in spans_of(lengths)] + [n], device="cuda")
    leaf = lp.clone().requires_grad_(True)
    ref = ref if kl_coef else None
    loss, stats = pt.policy_loss(leaf, None if on_policy else old, adv, t, ref_logps=ref, clip_low=0.2, clip_high=0.3, kl_coef=kl_coef,
                                 reduction=reduction, offsets=offsets)
    loss.backward()
    exact = torch.nan_to_num(lp.double()).requires_grad_(True)
    want, want_stats = ref_policy(exact, None if on_policy else torch.nan_to_num(old.double()), torch.nan_to_num(adv.double()),
                                  None if ref is None else torch.nan_to_num(ref.double()), t != IGNORE, spans_of(lengths), 0.2, 0.3, kl_coef, reduction)
    (grad,) = torch.autograd.grad(want, exact)
    # exp and expm1 in fp32 (2 units in the last place) on exact differences: 1e-6 of a token's terms, of size 1 here
    near(loss.detach().reshape(1), want.detach().reshape(1), 1e-6, 2e-6)
    near(stats, want_stats.detach(), 2e-6, 1e-7)
    near(leaf.grad, grad, 2e-6, 1e-6 * grad.abs().max().item())
    assert torch.all(leaf.grad[t == IGNORE] == 0)


def test_policy_with_nothing_counted_and_with_overflowing_ratios(pt):
    t = torch.full((2, 5), IGNORE, device="cuda")
    lp = torch.full((2, 5), math.nan, device="cuda").requires_grad_(True)
    for reduction in ("token", "sequence"):
        loss, stats = pt.policy_loss(lp, lp.detach(), torch.full((2, 5), math.nan, device="cuda"), t, ref_logps=lp.detach(), kl_coef=1.0,
                                     reduction=reduction)
        (grad,) = torch.autograd.grad(loss, lp)
        assert loss == 0 and torch.all(stats == 0) and torch.all(grad == 0)
    lp = torch.tensor([[-1.0, -1.0, -300.0]], device="cuda").requires_grad_(True)
    loss, stats = pt.policy_loss(lp, torch.tensor([[-200.0, -200.0, -1.0]], device="cuda"), torch.tensor([[1.0, 0.0, 1.0]], device="cuda"),
                                 torch.zeros(1, 3, dtype=torch.int64, device="cuda"))
    loss.backward()
    near(loss.detach().reshape(1), torch.tensor([-1.2 / 3], dtype=torch.float64, device="cuda"), 1e-6, 0)      # clipped; no advantage; ratio 0
    assert torch.all(lp.grad == 0)


def test_advantages_per_sequence(pt):
    lp = -torch.rand(4, 9, device="cuda", generator=gen(36))
    old = lp + 0.05
    adv = torch.randn(4, device="cuda", generator=gen(37))
    t = torch.zeros(4, 9, dtype=torch.int64, device="cuda")
    a = pt.policy_loss(lp, old, adv, t)[0]
    b = pt.policy_loss(lp, old, adv[:, None].expand(4, 9), t)[0]
    assert a == b
    with pytest.raises(Exception, match="sequences of one length"):
        pt.policy_loss(lp.view(-1), old.view(-1), adv, t.view(-1), offsets=torch.tensor([0, 9, 18, 27, 36], device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("vocab,cols,lengths", [(1000, 1024, [33, 33]), (777, 777, [1]), (50257, 50304, [20, 0, 41]), (50257, 50257, [3, 3]),
                                                (5000, 5001, [50, 7, 300]), (131000, 131000, [5]), (260000, 260008, [2, 1])])
def test_policy_loss_from_logits(pt, dtype, reduction, vocab, cols, lengths):
    rows = sum(lengths)
    x, t = logits_of(rows, vocab, cols, dtype, 41), targets_of(rows, vocab, 42)
    lp, probs, counted = ref_logps(x, t, vocab, 0.8)
    old, adv, ref = policy_inputs(lp, 43)
    exact = lp.clone().requires_grad_(True)
    want, want_stats = ref_policy(exact, old.double(), adv.double(), ref.double(), t != IGNORE, spans_of(lengths), 0.2, 0.3, 0.05, reduction)
    (row_grad,) = torch.autograd.grad(want, exact)
    dx = ref_dlogits(probs, counted, t, row_grad, cols, 0.8)
    offsets = torch.tensor([a for a, _ in spans_of(lengths)] + [rows], device="cuda")
    x[t == IGNORE] = math.nan
    loss_fn = pt.PolicyLoss(vocab, clip_low=0.2, clip_high=0.3, kl_coef=0.05, reduction=reduction, temperature=0.8, inplace=False)
    loss, stats, grad = loss_fn.loss_and_grad(x, (t, old, adv, ref), offsets=offsets, grad_scale=0.5)
    # the ratio carries the error of one log-probability
    err = 1e-6 * (1 + lp.abs().max().item())
    size = (row_grad.abs().max().item() + 1e-30)
    near(loss.reshape(1), want.detach().reshape(1), 2e-6, 2 * err)
    near(stats, want_stats.detach(), 2e-6, 2 * err)
    near(grad, 0.5 * dx, (4e-6 if dtype == torch.float32 else 2 ** -8) + 4 * err, 4 * err * size)
    assert torch.all(grad[:, vocab:] == 0) and torch.all(grad[t == IGNORE] == 0)
    with torch.no_grad():
        near(loss_fn(x, (t, old, adv, ref), offsets).reshape(1), loss.double().reshape(1), 1e-6, 2 * err)
    # autograd: the gradient is made in the forward call, for grad_scale; another upstream gradient rescales it
    loss_fn.grad_scale = 0.5
    for upstream in (0.5, 0.25):
        leaf = x.clone().requires_grad_(True)
        (loss_fn(leaf, (t, old, adv, ref), offsets) * upstream).backward()
        if upstream == 0.5:
            assert torch.equal(leaf.grad, grad)
        else:
            near(leaf.grad, 0.5 * grad.double(), 2 ** -8 if dtype == torch.bfloat16 else 2 ** -23, 1e-38)
    over = x.clone()
    assert torch.equal(loss_fn.loss_and_grad(over, (t, old, adv, ref), offsets=offsets, out=over, grad_scale=0.5)[2], grad)


# Rows that 32, 64, 128, 256 and 512 threads work on (the last for gradients)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,cols", [(4100, 1000, 1003), (2100, 5001, 5001), (1100, 12001, 12008), (700, 12001, 12001), (2050, 41003, 41003)])
def test_many_rows_of_every_size(pt, rows, vocab, cols, dtype):
    x, t = logits_of(rows, vocab, cols, dtype, 61), targets_of(rows, vocab, 62)
    t[:2] = 7
    x[0, :vocab] = torch.finfo(dtype).min
    x[1, :vocab] = -math.inf
    g = torch.randn(rows, device="cuda", generator=gen(63))
    lp, probs, counted = ref_logps(x, t, vocab, 0.9)
    want = ref_dlogits(probs, counted, t, g, cols, 0.9)
    lp[1], want[1] = -math.inf, 0.0
    leaf = x.clone().requires_grad_(True)
    out = pt.token_logprobs(leaf, t, vocab, temperature=0.9)
    near(out.detach(), lp, 1e-6, 1e-6)
    near(pt.token_logprobs(x, t, vocab, temperature=0.9), lp, 1e-6, 1e-6)
    out.backward(g)
    near(leaf.grad, want, 4e-6 if dtype == torch.float32 else 2 ** -8, 1e-7 * g.abs().max().item() / 0.9)
    del leaf, want
    # the policy loss on all but the first two
    t[:2] = IGNORE
    counted[:2] = False
    lp[:2] = 0.0
    old, adv, ref = policy_inputs(lp, 64)
    exact = lp.clone().requires_grad_(True)
    loss, _ = ref_policy(exact, old.double(), adv.double(), ref.double(), t != IGNORE, spans_of([rows]), 0.2, 0.3, 0.05, "token")
    (row_grad,) = torch.autograd.grad(loss, exact)
    err, size = 1e-6 * (1 + lp.abs().max().item()), row_grad.abs().max().item()
    loss_fn = pt.PolicyLoss(vocab, clip_low=0.2, clip_high=0.3, kl_coef=0.05, temperature=0.9, inplace=False)
    got, _, grad = loss_fn.loss_and_grad(x, (t, old, adv, ref), offsets=torch.tensor([0, rows], device="cuda"))
    near(got.reshape(1), loss.detach().reshape(1), 2e-6, 2 * err)
    near(grad, ref_dlogits(probs, counted, t, row_grad, cols, 0.9), (4e-6 if dtype == torch.float32 else 2 ** -8) + 4 * err, 4 * err * size)


@pytest.mark.parametrize("rows,vocab,dtype", [(2050, 41003, torch.bfloat16), (3000, 50257, torch.bfloat16), (1100, 12001, torch.float32)])
def test_policy_rows_wait_for_their_readers(pt, rows, vocab, dtype):
    """Rows that follow one another through shared memory: the same result every time."""
    x, t = logits_of(rows, vocab, vocab, dtype, 71), targets_of(rows, vocab, 72)
    old, adv, ref = policy_inputs(pt.token_logprobs(x, t).double(), 73)
    loss_fn = pt.PolicyLoss(vocab, clip_low=0.2, clip_high=0.3, kl_coef=0.05, temperature=0.9, inplace=False)
    offsets, first = torch.tensor([0, rows], device="cuda"), None
    for _ in range(25):
        loss, stats, grad = loss_fn.loss_and_grad(x, (t, old, adv, ref), offsets=offsets)
        assert first is None or (torch.equal(grad, first[2]) and torch.equal(stats, first[1]) and loss == first[0])
        first = first or (loss, stats, grad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("vocab", [1003, 30011])
def test_losses_on_rows_that_start_anywhere(pt, vocab, offset, dtype):
    """Windows of a wider matrix: gradients beside them (another alignment) and over them, with nothing around touched."""
    rows, ld = 24, vocab + 18
    whole = logits_of(rows, ld, ld, dtype, 45)
    x, t = whole[:, offset:offset + vocab], targets_of(rows, vocab, 46)
    lp, _, _ = ref_logps(x, t, vocab)
    old, adv, ref = policy_inputs(lp, 47)
    offsets = torch.tensor([0, 5, 12, 13, 24], device="cuda")
    for fn, labels in ((pt.PolicyLoss(vocab, clip_high=0.3, kl_coef=0.05), (t, old, adv, ref)), (pt.PreferenceLoss(vocab), (t, ref))):
        loss, extra, want = fn.loss_and_grad(x.contiguous(), labels, offsets=offsets)
        beside = fn.loss_and_grad(x, labels, offsets=offsets)
        near(beside[0].reshape(1), loss.double().reshape(1), 1e-6, 1e-6)
        # (rows that start elsewhere are summed in another order: a unit or two in the last place of the sums)
        near(beside[2], want.double(), 2 ** -7 if dtype == torch.bfloat16 else 4e-6, 1e-7)
        over = whole.clone()
        got = fn.loss_and_grad(over[:, offset:offset + vocab], labels, offsets=offsets, out=over[:, offset:offset + vocab])[2]
        assert torch.equal(got, beside[2])
        assert torch.equal(over[:, :offset], whole[:, :offset]) and torch.equal(over[:, offset + vocab:], whole[:, offset + vocab:])


def test_more_than_two_to_the_31_logits(pt):
    rows, vocab, cols = 43000, 50257, 50304
    x = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    x[:-3] = 0
    x[-3:] = logits_of(3, cols, cols, torch.bfloat16, 48)
    t = torch.full((rows,), IGNORE, device="cuda")
    t[-3:] = torch.tensor([50256, 0, 777], device="cuda")
    tail = x[-3:].clone()
    lp, probs, counted = ref_logps(tail, t[-3:], vocab)
    near(pt.token_logprobs(x, t, vocab)[-3:], lp, 1e-6, 1e-6)
    fn = pt.PolicyLoss(vocab, inplace=True)
    labels = (t.view(1, -1), None, torch.ones(rows, device="cuda").view(1, -1))
    loss, _, grad = fn.loss_and_grad(x.view(1, rows, cols), labels, out=x.view(1, rows, cols))
    near(loss.reshape(1), torch.tensor([-1.0], dtype=torch.float64, device="cuda"), 1e-6, 0)
    want = ref_dlogits(probs, counted, t[-3:], torch.full((3,), -1 / 3, device="cuda"), cols)
    near(grad[0, -3:], want, 2 ** -8, 1e-7)
    assert torch.all(x[:-3] == 0)


# ----------------------------------------------------------------------------------- gradient norm and clipping
def grad_list(sizes, dtypes, seed, scale=1.0):
    return [(torch.randn(n, device="cuda", generator=gen(seed + i)) * scale).to(d) for i, (n, d) in enumerate(zip(sizes, dtypes))]


@pytest.mark.parametrize("sizes", [[1], [7, 1, 4097], [5_000_003], [100] * 300, [65536, 3, 200_000, 8, 1_000_001]], ids=lambda s: str(s)[:30])
@pytest.mark.parametrize("dtypes", ["fp32", "bf16", "mixed"])
def test_clip_grad_norm(pt, sizes, dtypes):
    kinds = {"fp32": [torch.float32], "bf16": [torch.bfloat16], "mixed": [torch.float32, torch.bfloat16]}[dtypes]
    grads = grad_list(sizes, [kinds[i % len(kinds)] for i in range(len(sizes))], 51)
    before = [g.clone() for g in grads]
    norm = torch.sqrt(sum(g.double().square().sum() for g in grads))
    near(pt.global_grad_norm(grads).reshape(1), norm.reshape(1), 1e-6, 0)
    near(pt.clip_grad_norm_(grads, 1e9).reshape(1), norm.reshape(1), 1e-6, 0)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))              # within the norm: untouched
    limit = 0.3 * norm.item()
    near(pt.clip_grad_norm_(grads, limit).reshape(1), norm.reshape(1), 1e-6, 0)
    coef = limit / (norm + 1e-6)
    for g, b in zip(grads, before):
        near(g, b.double() * coef, 2 ** -8 if g.dtype == torch.bfloat16 else 1e-6, 0)


def test_clip_of_views_parameters_and_odd_starts(pt):
    base = torch.randn(1001, device="cuda", generator=gen(61))
    table = torch.randn(64, 48, device="cuda", generator=gen(62)).bfloat16()
    p = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    p.grad = torch.arange(5.0, device="cuda")
    q = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    q.main_grad = torch.full((3,), 2.0, device="cuda")
    unused = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    views = [base[1:778], table[:, 3:40], table.t()[40:44], torch.zeros(0, device="cuda"), p, q, unused]
    old = [v.detach().clone() for v in views[:3]]
    norm = torch.sqrt(sum(v.double().square().sum() for v in [*old, p.grad, q.main_grad]))
    outside = (base[:1].clone(), base[778:].clone(), table[:, :3].clone())
    near(pt.clip_grad_norm_(views, 0.5).reshape(1), norm.reshape(1), 1e-6, 0)
    coef = 0.5 / (norm + 1e-6)
    for v, o in zip(views[:3], old):
        near(v, o.double() * coef, 2 ** -8 if v.dtype == torch.bfloat16 else 1e-6, 0)
    near(p.grad, torch.arange(5.0, device="cuda").double() * coef, 1e-6, 0)
    near(q.main_grad, torch.full((3,), 2.0, device="cuda").double() * coef, 1e-6, 0)
    assert torch.equal(base[:1], outside[0]) and torch.equal(base[778:], outside[1]) and torch.equal(table[:, :3], outside[2])
    assert pt.clip_grad_norm_([], 1.0) == 0 and pt.clip_grad_norm_([unused], 1.0) == 0


def test_clip_of_infinite_and_missing_gradients(pt):
    g = torch.ones(1000, device="cuda")
    g[3] = math.nan
    assert torch.isnan(pt.clip_grad_norm_([g], 1.0)) and torch.isnan(g).all()
    g = torch.ones(1000, device="cuda")
    g[3] = math.inf
    assert pt.clip_grad_norm_([g], 1.0) == math.inf and g[0] == 0 and torch.isnan(g[3])
    g = torch.zeros(1000, device="cuda")
    assert pt.clip_grad_norm_([g], 1.0) == 0 and torch.all(g == 0)


@pytest.mark.parametrize("adam_w", [True, False])
@pytest.mark.parametrize("n", [4, 1000, 4_000_004])
def test_adam_step_clipped(pt, n, adam_w):
    state = [torch.randn(n, device="cuda", generator=gen(71 + i)) for i in range(3)] + [torch.rand(n, device="cuda", generator=gen(75))]
    for limit, grad_scale in ((0.2 * math.sqrt(n), 1.0), (1e9, 0.5)):
        p, g, m, v = (s.clone() for s in state)
        lp = p.bfloat16()
        norm = pt.adam_step_clipped(p, g, m, v, lp, max_norm=limit, lr=1e-2, step=3, weight_decay=0.1, adam_w_mode=adam_w, grad_scale=grad_scale)
        P, G, M, V = (s.double() for s in state)
        want_norm = grad_scale * G.norm()
        G = G * grad_scale * min(1.0, limit / (want_norm.item() + 1e-6))
        if not adam_w:
            G = G + 0.1 * P
        M, V = 0.9 * M + 0.1 * G, 0.999 * V + 0.001 * G * G
        step = (M / (1 - 0.9 ** 3)) / ((V / (1 - 0.999 ** 3)).sqrt() + 1e-8) + (0.1 * P if adam_w else 0)
        P = P - 1e-2 * step
        near(norm.reshape(1), want_norm.reshape(1), 1e-6, 0)
        near(m, M, 1e-6, 1e-6)
        near(v, V, 1e-6, 0)
        near(p, P, 1e-6, 1e-6 * step.abs().max().item())
        assert torch.equal(lp, p.bfloat16()) and torch.all(g == 0)


def test_streams_and_repeats(pt):
    """The same call on another stream than the one its inputs were made on, and again: the same bits."""
    x, t = logits_of(64, 5000, 5000, torch.bfloat16, 81), targets_of(64, 5000, 82)
    fn = pt.PolicyLoss(5000, inplace=False)
    lp = pt.token_logprobs(x, t)
    labels = (t.view(4, 16), lp.view(4, 16) + 0.01, torch.ones(4, device="cuda"))
    a = fn.loss_and_grad(x.view(4, 16, -1), labels)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = fn.loss_and_grad(x.view(4, 16, -1), labels)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    grads = grad_list([100_000, 333], [torch.float32, torch.bfloat16], 83)
    assert pt.global_grad_norm(grads) == pt.global_grad_norm(grads)


# ----------------------------------------------------------------------------------- refusals
def test_refusals(pt):
    from bamboo_b200 import lib
    x, t = logits_of(4, 10, 16, torch.float32, 91), torch.zeros(4, dtype=torch.int64, device="cuda")
    for vocab in (0, 17, -1):
        with pytest.raises(ValueError):
            pt.token_logprobs(x, t, vocab)
    with pytest.raises(ValueError):
        pt.token_logprobs(x, t[:3])
    with pytest.raises(ValueError):
        pt.token_logprobs(x, t, temperature=0.0)
    with pytest.raises(TypeError):
        pt.token_logprobs(x, t.float())
    with pytest.raises(lib.BambooNativeError):
        pt.token_logprobs(x.half(), t)
    with pytest.raises(lib.BambooNativeError):
        pt.token_logprobs(x, t.cpu())
    lp = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="pairs"):
        pt.preference_loss(lp[:3].view(3, 1), None, t[:3].view(3, 1))
    with pytest.raises(ValueError):
        pt.preference_loss(lp, None, t)
    with pytest.raises(ValueError):
        pt.preference_loss(lp.view(2, 2), None, t.view(2, 2), form="cubic")
    for bad in ({"beta": 0.0}, {"label_smoothing": 1.5}):
        with pytest.raises(lib.BambooNativeError):
            pt.preference_loss(lp.view(2, 2), None, t.view(2, 2), **bad)
    with pytest.raises(ValueError):
        pt.policy_loss(lp.view(2, 2), None, lp, t.view(2, 2), reduction="mean")
    with pytest.raises(ValueError):
        pt.policy_loss(lp.view(2, 2), lp[:2], lp, t.view(2, 2))
    for bad in ({"clip_low": -0.1}, {"kl_coef": -1.0}):
        with pytest.raises(lib.BambooNativeError):
            pt.policy_loss(lp.view(2, 2), None, lp, t.view(2, 2), **bad)
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError):
            pt.clip_grad_norm_([lp], bad)
    with pytest.raises(lib.BambooNativeError):
        pt.clip_grad_norm_([lp.half()], 1.0)
    with pytest.raises(lib.BambooNativeError):
        pt.clip_grad_norm_([lp, lp.cpu()], 1.0)
    shifted = torch.zeros(5, 16, device="cuda")
    with pytest.raises(lib.BambooNativeError, match="overlaps"):
        pt.PreferenceLoss(10).loss_and_grad(shifted[:4].view(2, 2, 16), (t.view(2, 2), None), out=shifted[1:].view(2, 2, 16))
    torch.cuda.synchronize()


def test_offsets_that_do_not_ascend_are_reported(pt):
    from bamboo_b200 import lib
    lp, t = torch.zeros(8, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")
    for offsets in ([0, 5, 3], [-4, 2, 8], [0, 4, 9], [6, 1 << 40, 8]):
        off = torch.tensor(offsets, device="cuda")
        pt.preference_loss(lp, lp, t, offsets=off)
        torch.cuda.synchronize()
        assert lib.read_status() < 0
        pt.policy_loss(lp, lp, lp, t, offsets=off, reduction="sequence")
        torch.cuda.synchronize()
        assert lib.read_status() < 0


def test_gradient_clipping_in_a_graph_beside_other_calls(pt):
    """A captured norm replayed between calls that are launched one by one: counters of their own, the same results."""
    grads = [torch.randn(n, device="cuda", generator=gen(200 + n)) for n in (70001, 5, 300000)]
    want = torch.sqrt(sum(g.double().square().sum() for g in grads))
    keep, other = [g.clone() for g in grads], [torch.ones(50000, device="cuda")]
    pt.global_grad_norm(grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = pt.clip_grad_norm_(grads, 0.25)
    for _ in range(4):
        for g, k in zip(grads, keep):
            g.copy_(k)
        graph.replay()
        near(pt.global_grad_norm(other).reshape(1), torch.tensor([50000 ** 0.5], dtype=torch.float64, device="cuda"), 1e-6, 0)
        near(norm.reshape(1), want.reshape(1), 1e-6, 0)
        for g, k in zip(grads, keep):
            near(g, k.double() * (0.25 / (want + 1e-6)), 1e-6, 0)

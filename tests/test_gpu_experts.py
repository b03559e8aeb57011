"""Routing, moving rows to experts and back, and the experts' products against their definitions in 64 bits: sizes, strides and masks where
they can go wrong, gradients against the formula's and against differences, a whole mixture as it is used, and captured calls.

Tolerances follow from the arithmetic.  Routing: a probability is a quotient of ex2-based exponentials (2^-22 each for arguments below 64: the argument's
rounding, 2^-24 x 64, and the function's two units) and a sum of up to 256 of them in 32 bits: 2e-5 relative covers it; the gradient subtracts such
products from each other, so its floor is 2e-5 of the largest term.  Moved rows are copies; sums of k rows take k + 1 roundings of 2^-24 of the
absolute terms and one to the output's type (half a step: 2^-8 bf16).  Products: bf16 products are exact in fp32, each of the K additions in the tensor
core may truncate, 2^-23 of the absolute sum, and the output is rounded once, 2^-8; chains propagate these bounds in 64 bits (``Bound``)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2 ** -8, FP32: 2 ** -24}


@pytest.fixture(scope="module")
def ex():
    from bamboo_b200 import experts, lib
    lib.load()
    lib.read_status()
    return experts


@pytest.fixture(autouse=True)
def healthy():
    yield
    from bamboo_b200 import lib
    torch.cuda.synchronize()
    assert lib.read_status() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=FP32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen(seed)) * scale).to(dtype)


def near(got, want, rel, floor=0.0):
    """|got - want| <= rel |want| + floor, with NaN and infinities in the same places."""
    assert got.shape == want.shape
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    finite = torch.isfinite(want)
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
    floor = torch.as_tensor(floor, device=want.device, dtype=torch.float64).expand(want.shape)
    over = ((got - want).abs() - rel * want.abs() - floor)[finite]
    assert not (over > 0).any(), (over.max().item(), want[finite].abs().max().item())


# ----------------------------------------------------------------------------------- routing
def ref_route(logits, k, n, normalize):
    """64-bit routing with autograd, as a dict; whole-number parts without a sort."""
    x = logits[:, :n].double()
    t = x.shape[0]
    left = x.detach().clone()
    picks = []
    for _ in range(k):
        value = torch.where(left.isnan(), math.inf, left)
        first_nan = left.isnan().any(1)
        best = torch.where(first_nan, left.isnan().int().argmax(1), value.argmax(1))
        ok = first_nan | (value.max(1).values > -math.inf)
        picks.append(torch.where(ok, best, -1))
        left[torch.arange(t, device="cuda"), best] = -math.inf
    chosen = torch.stack(picks, 1)
    alive = chosen[:, 0] >= 0
    member = torch.zeros(t, n + 1, dtype=torch.bool, device="cuda").scatter_(1, torch.where(chosen < 0, n, chosen), True)[:, :n]
    probs = torch.zeros_like(x)
    probs[alive] = torch.softmax(x[alive], 1)
    base = probs
    if normalize:
        base = torch.zeros_like(x)
        base[alive] = torch.softmax(x.masked_fill(~member, -math.inf)[alive], 1)
    weights = torch.where(chosen >= 0, base.gather(1, chosen.clamp(min=0)), 0.0)
    count = member.sum(0)
    balance = n * torch.dot(count / count.sum().clamp(min=1).double(), probs.sum(0) / alive.sum().clamp(min=1))
    flat = chosen.reshape(-1)
    rows, slots, at, starts = torch.full_like(flat, -1), torch.full_like(flat, -1), 0, [0]
    for e in range(n):
        mine = (flat == e).nonzero()[:, 0]
        rows[mine] = torch.arange(at, at + len(mine), device="cuda")
        slots[at:at + len(mine)] = mine
        at += len(mine)
        starts.append(at)
    return {"weights": weights, "experts": chosen, "rows": rows.view_as(chosen), "slots": slots, "offsets": torch.tensor(starts, device="cuda"),
            "balance": balance}


def check_route(r, want, rel=2e-5):
    for name in ("experts", "rows", "slots", "offsets"):
        got = getattr(r, name)
        assert got.dtype == torch.int32 and torch.equal(got.long().view_as(want[name]), want[name]), name
    near(r.weights.detach().view_as(want["weights"]), want["weights"].detach(), rel)
    near(r.balance.detach(), want["balance"].detach(), rel)


ROUTES = [(1, 1, 1, 1), (1, 8, 8, 2), (7, 2, 2, 2), (33, 5, 8, 3), (512, 8, 8, 2), (1000, 31, 32, 4), (257, 33, 33, 8), (2500, 64, 64, 6), (300, 65, 72, 1),
          (129, 128, 128, 8), (90, 200, 200, 5), (4801, 256, 256, 8), (40, 256, 260, 32), (700, 12, 12, 12), (9000, 3, 3, 1)]


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens,experts,cols,k", ROUTES)
def test_route_and_gradient(ex, tokens, experts, cols, k, dtype, normalize):
    x = randn(tokens, cols, seed=tokens + experts, scale=2.0).to(dtype)       # (bf16: ties among many experts)
    masked = torch.rand(tokens, device="cuda", generator=gen(3)) < 0.1
    x[masked] = -math.inf
    x[torch.rand(tokens, cols, device="cuda", generator=gen(4)) < 0.1] = -math.inf
    check_route(ex.route(x, k, experts, normalize=normalize), ref_route(x, k, experts, normalize))
    leaf, exact = x.clone().requires_grad_(True), x.double().requires_grad_(True)
    r, want = ex.route(leaf, k, experts, normalize=normalize), ref_route(exact, k, experts, normalize)
    check_route(r, want)
    dw, db = randn(tokens, k, seed=5), torch.tensor(0.7, device="cuda")
    for a, b in ((dw, db), (dw, None), (None, db)):
        outs = [(r.weights, want["weights"], a), (r.balance, want["balance"], b)]
        outs = [o for o in outs if o[2] is not None]
        (got,) = torch.autograd.grad([o[0] for o in outs], leaf, [o[2] for o in outs], retain_graph=True)
        (ref,) = torch.autograd.grad([o[1] for o in outs], exact, [o[2].double() for o in outs], retain_graph=True)
        ref = torch.nan_to_num(ref)              # (64-bit softmax of rows that the reference leaves out: 0)
        scale = (0 if a is None else a.abs().max().item() * 2) + (0 if b is None else experts * 0.7 * 2 / tokens)
        near(got, ref, HALF_STEP[dtype] + 2e-5, 2e-5 * scale)
        assert torch.all(got[:, experts:] == 0)


@pytest.mark.parametrize("tokens,experts,cols,k", [(t + more, e, c, k) for t, e, c, k in ((128, 8, 8, 2), (128, 17, 24, 8), (64, 64, 64, 16), (32, 129, 129, 8))
                                                   for more in (-1, 0, 1)])
def test_route_by_one_block_and_by_several(ex, tokens, experts, cols, k):
    test_route_and_gradient(ex, tokens, experts, cols, k, FP32, True)
    none = ex.route(torch.full((tokens, experts), -math.inf, device="cuda"), k)
    assert torch.all(none.rows == -1) and torch.all(none.slots == -1) and torch.all(none.offsets == 0) and torch.all(none.weights == 0)


def test_route_ties_go_to_the_lower_index(ex):
    x = torch.zeros(70, 40, device="cuda")
    x[1::2, 7], x[1::2, 30], x[::3, 2] = 1.0, 1.0, -0.0
    check_route(ex.route(x, 3), ref_route(x + 0.0, 3, 40, True))
    assert ex.route(x, 3).experts[0].tolist() == [0, 1, 2] and ex.route(x, 3).experts[1].tolist() == [7, 30, 0]


def test_route_values_out_of_the_ordinary(ex):
    """NaN above all, infinities, the types' lowest values, rows without anything to choose, fewer than k to choose."""
    inf, nan, low = math.inf, math.nan, torch.finfo(FP32).min
    x = torch.tensor([[0.0, 1.0, -inf, -inf], [-inf] * 4, [low, low, -inf, low], [-inf, -inf, -inf, 3.0], [1e30, -1e30, 0, 1e30], [0.0, nan, 2.0, -inf],
                      [5.0, inf, 1.0, 2.0], [88.0, -88.0, 0.0, 87.5]], device="cuda")
    for normalize in (True, False):
        r = ex.route(x, 3, normalize=normalize)
        want = ref_route(x, 3, 4, normalize)
        for name in ("experts", "rows", "slots", "offsets"):
            assert torch.equal(getattr(r, name).long().view_as(want[name]), want[name]), name
        near(r.weights[[0, 1, 2, 3, 4, 7]], want["weights"][[0, 1, 2, 3, 4, 7]], 2e-5, 1e-37)
        assert r.weights[5:7, 0].isnan().all() and r.weights[1].tolist() == [0.0] * 3
    clean = x[[0, 1, 2, 3, 4, 7]].clone().requires_grad_(True)
    r = ex.route(clean, 3)
    (g,) = torch.autograd.grad((r.weights, r.balance), clean, (torch.ones_like(r.weights), torch.tensor(1.0, device="cuda")))
    assert torch.isfinite(g).all() and torch.all(g[1] == 0)
    nothing = ex.route(torch.full((9, 5), -inf, device="cuda"), 2)
    assert torch.all(nothing.offsets == 0) and torch.all(nothing.slots == -1) and torch.all(nothing.rows == -1) and nothing.balance == 0


def test_route_shapes_and_strides(ex):
    x = randn(6 * 5, 24, seed=9)
    want = ref_route(x, 3, 20, True)
    r = ex.route(x.view(6, 5, 24), 3, 20)
    assert r.weights.shape == r.experts.shape == r.rows.shape == (6, 5, 3)
    check_route(r, want)
    wide = randn(30, 61, seed=10)
    wide[:, 5:29] = x
    check_route(ex.route(wide[:, 5:29], 3, 20), want)
    check_route(ex.route(x.t().contiguous().t(), 3, 20), want)
    leaf = wide.clone().requires_grad_(True)
    r = ex.route(leaf[:, 5:29], 3, 20)
    dw = randn(30, 3, seed=11)
    (g,) = torch.autograd.grad(r.weights, leaf, dw)
    whole = x.clone().requires_grad_(True)
    (w,) = torch.autograd.grad(ex.route(whole, 3, 20).weights, whole, dw)
    assert torch.equal(g[:, 5:29], w) and torch.all(g[:, :5] == 0) and torch.all(g[:, 29:] == 0)
    none = ex.route(x[:0], 3, 20)
    assert none.weights.shape == (0, 3) and none.offsets.tolist() == [0] * 21 and none.balance == 0
    empty = x[:0].clone().requires_grad_(True)
    r = ex.route(empty, 3, 20)
    assert torch.autograd.grad(r.weights.sum() + r.balance, empty)[0].shape == (0, 24)


def test_route_gradient_against_differences(ex):
    x = randn(11, 9, seed=12)
    dw, leaf = randn(11, 4, seed=13), x.clone().requires_grad_(True)
    r = ex.route(leaf, 4, normalize=False)
    (g,) = torch.autograd.grad((r.weights * dw).sum() + 3 * r.balance, leaf)
    for i, j in ((0, 0), (3, 8), (10, 4), (7, 2)):
        step = 1e-3
        up, down = x.clone(), x.clone()
        up[i, j] += step
        down[i, j] -= step
        a, b = (ex.route(z, 4, normalize=False) for z in (up, down))
        assert torch.equal(a.experts, r.experts) and torch.equal(b.experts, r.experts)        # (the choice stays)
        slope = ((a.weights - b.weights).double() * dw.double()).sum() + 3 * (a.balance - b.balance).double()
        # 32-bit differences over a step of 2e-3: 4 values of 2^-23 and a balance of about 1
        assert abs(slope / (2 * step) - g[i, j]) < 2e-3


# ----------------------------------------------------------------------------------- rows there and back
def routing_of(ex, tokens, experts, k, seed, masked=0.15):
    x = randn(tokens, experts, seed=seed)
    x[torch.rand(tokens, device="cuda", generator=gen(seed + 1)) < masked] = -math.inf
    x[torch.rand(tokens, experts, device="cuda", generator=gen(seed + 2)) < 0.2] = -math.inf
    return ex.route(x, k, normalize=False)


MOVES = [(1, 8, 1, 1), (7, 1024, 8, 2), (300, 256, 8, 2), (65, 1, 4, 3), (40, 77, 5, 4), (500, 1000, 64, 8), (33, 4104, 8, 2), (3, 16392, 4, 2), (9, 20001, 3, 3),
         (1200, 2048, 6, 1), (2, 8, 32, 32)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens,hidden,experts,k", MOVES)
def test_dispatch_and_combine(ex, tokens, hidden, experts, k, dtype):
    r = routing_of(ex, tokens, experts, k, 21)
    x, dout = randn(tokens, hidden, seed=22, dtype=dtype), randn(tokens * k, hidden, seed=23, dtype=dtype)
    slots, rows = r.slots.long(), r.rows.long()
    want = torch.where((slots >= 0)[:, None], x[slots.clamp(min=0) // k], torch.zeros((), device="cuda", dtype=dtype))
    assert torch.equal(ex.dispatch(x, r), want)
    leaf = x.clone().requires_grad_(True)
    y = ex.dispatch(leaf, r)
    assert torch.equal(y.detach(), want)
    (dx,) = torch.autograd.grad(y, leaf, dout)
    each = torch.where((rows >= 0)[:, :, None], dout.double()[rows.clamp(min=0)], 0.0)
    near(dx, each.sum(1), HALF_STEP[dtype], (k + 1) * 2 ** -24 * each.abs().sum(1))

    xs, res, dy = randn(tokens * k, hidden, seed=24, dtype=dtype), randn(tokens, hidden, seed=25, dtype=dtype), randn(tokens, hidden, seed=26, dtype=dtype)
    xs[r.offsets[-1]:] = math.nan                                      # nobody's rows
    each = torch.where((rows >= 0)[:, :, None], xs.double()[rows.clamp(min=0)], 0.0)
    terms = r.weights.double()[:, :, None] * each
    for residual in (None, res):
        out = terms.sum(1) + (0 if residual is None else residual.double())
        floor = (k + 2) * 2 ** -24 * (terms.abs().sum(1) + (0 if residual is None else residual.double().abs()))
        near(ex.combine(xs, r, residual=residual), out, HALF_STEP[dtype], floor)
        a, w, c = xs.clone().requires_grad_(True), r.weights.clone().requires_grad_(True), None if residual is None else residual.clone().requires_grad_(True)
        y = ex.combine(a, r._replace(weights=w), residual=c)
        near(y.detach(), out, HALF_STEP[dtype], floor)
        grads = torch.autograd.grad(y, [a, w] + ([] if c is None else [c]), dy)
        at = slots.clamp(min=0)
        dxs = torch.where((slots >= 0)[:, None], r.weights.double().reshape(-1)[at][:, None] * dy.double()[at // k], 0.0)
        near(grads[0], dxs, HALF_STEP[dtype] + 2 ** -24)
        products = each * dy.double()[:, None]
        # a thread adds at most hidden / 32 + 16 products one after the other, then come five sums a run and the runs: below hidden / 16 + 16 roundings
        near(grads[1], products.sum(2), 2 ** -24, (hidden / 16 + 16) * 2 ** -24 * products.abs().sum(2))
        if c is not None:
            assert torch.equal(grads[2], dy)
    only = r.weights.clone().requires_grad_(True)                      # weights alone, rows alone
    (dw,) = torch.autograd.grad(ex.combine(xs, r._replace(weights=only)), only, dy)
    assert torch.equal(dw, grads[1])
    rows_only = xs.clone().requires_grad_(True)
    (da,) = torch.autograd.grad(ex.combine(rows_only, r), rows_only, dy)
    assert torch.equal(da, grads[0])


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_moved_rows_of_other_strides(ex, dtype):
    tokens, k, h = 50, 2, 96
    r = routing_of(ex, tokens, 8, k, 31)
    wide = randn(tokens, 131, seed=32, dtype=dtype)
    for offset in (0, 1, 3, 8):
        part = wide[:, offset:offset + h]
        whole = part.contiguous()
        assert torch.equal(ex.dispatch(part, r), ex.dispatch(whole, r))
        xs = randn(tokens * k, 131, seed=33, dtype=dtype)[:, offset:offset + h]
        assert torch.equal(ex.combine(xs, r, residual=part), ex.combine(xs.contiguous(), r, residual=whole))
        leaf = wide.clone().requires_grad_(True)
        dout = randn(131, tokens * k, seed=34, dtype=dtype).t()[:, offset:offset + h]           # a gradient that arrives turned
        (g,) = torch.autograd.grad(ex.dispatch(leaf[:, offset:offset + h], r), leaf, dout)
        other = whole.clone().requires_grad_(True)
        (w,) = torch.autograd.grad(ex.dispatch(other, r), other, dout.contiguous())
        assert torch.equal(g[:, offset:offset + h], w)
    x3 = randn(5, 10, h, seed=35, dtype=dtype)
    r3 = r._replace(weights=r.weights.view(5, 10, k), rows=r.rows.view(5, 10, k), experts=r.experts.view(5, 10, k))
    assert torch.equal(ex.dispatch(x3, r3), ex.dispatch(x3.view(50, h), r))
    assert torch.equal(ex.combine(xs, r3), ex.combine(xs, r).view(5, 10, h))
    assert torch.equal(ex.dispatch(x3.transpose(0, 1).contiguous().transpose(0, 1), r3), ex.dispatch(x3, r3))
    none = ex.route(randn(0, 8), 2)
    assert ex.dispatch(randn(0, h, dtype=dtype), none).shape == (0, h) and ex.combine(randn(0, h, dtype=dtype), none).shape == (0, h)


def test_indexes_that_point_nowhere_are_left_out(ex):
    from bamboo_b200 import lib
    r = routing_of(ex, 20, 4, 2, 41, masked=0.0)
    x, xs = randn(20, 64, seed=42), randn(40, 64, seed=43)
    bad = r.slots.clone()
    bad[3], bad[5] = 40, -7
    y = ex.dispatch(x, r._replace(slots=bad))
    torch.cuda.synchronize()
    assert lib.read_status() == -1
    assert torch.all(y[3] == 0) and torch.all(y[5] == 0)
    rows = r.rows.clone()
    rows[2, 1] = 40
    got = ex.combine(xs, r._replace(rows=rows))
    torch.cuda.synchronize()
    assert lib.read_status() == -1
    rows[2, 1] = -1
    assert torch.equal(got, ex.combine(xs, r._replace(rows=rows)))
    assert lib.read_status() == 0


@pytest.mark.parametrize("hidden", [64, 77, 4104])
def test_choices_dropped_by_their_place(ex, hidden):
    """-1 in ``rows`` alone: the row that stays behind has a gradient of zeros, whatever lay in its memory."""
    r = routing_of(ex, 40, 4, 2, 44)
    rows = r.rows.clone()
    rows[5:25, 1] = -1
    r = r._replace(rows=rows)
    places = rows[rows >= 0].long()
    xs, dy = randn(80, hidden, seed=45).requires_grad_(True), randn(40, hidden, seed=46)
    y = ex.combine(xs, r)
    junk = [torch.full((80, hidden), math.nan, device="cuda") for _ in range(4)]
    del junk
    (dxs,) = torch.autograd.grad(y, xs, dy)
    want = torch.zeros(80, hidden, dtype=torch.float64, device="cuda")
    want[places] = (r.weights.double()[:, :, None] * dy.double()[:, None])[rows >= 0]
    near(dxs, want, 2 ** -23)


def test_places_that_name_another_slot_are_left_out(ex):
    from bamboo_b200 import lib
    r = routing_of(ex, 20, 4, 2, 47, masked=0.0)
    rows = r.rows.clone()
    there = rows >= 0
    a, b = rows[there].long()[:2].tolist()                              # two slots at one place
    rows[rows == b] = a
    xs, dy = randn(40, 64, seed=48).requires_grad_(True), randn(20, 64, seed=49)
    (dxs,) = torch.autograd.grad(ex.combine(xs, r._replace(rows=rows)), xs, dy)
    torch.cuda.synchronize()
    assert lib.read_status() == -1
    (want,) = torch.autograd.grad(ex.combine(xs, r), xs, dy)
    assert torch.all(dxs[b] == 0)
    want[b] = 0
    assert torch.equal(dxs, want)


# ----------------------------------------------------------------------------------- products
class Bound:
    """A value in 64 bits with a bound on how far the kernels' may be from it."""

    def __init__(self, value, err=0.0):
        self.value, self.err = value, torch.as_tensor(err, dtype=torch.float64, device="cuda").expand(value.shape)

    def rounded(self, dtype=BF16):
        return Bound(self.value, self.err + HALF_STEP[dtype] * (self.value.abs() + self.err))

    def check(self, got):
        near(got, self.value, 0.0, self.err)


def matmul(a, b):
    """a @ b of bounds, one summation in the tensor core."""
    size = a.value.abs() + a.err
    value = a.value @ b.value
    err = a.err @ (b.value.abs() + b.err) + size @ b.err + a.value.shape[-1] * 2 ** -23 * (size @ (b.value.abs() + b.err))
    return Bound(value, err)


def offsets_of(lengths, before=0):
    out = [before]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda"), out


def per_expert(fn, lengths, before, *tensors):
    """[(expert, fn of its rows)] over experts with rows"""
    at, out = before, []
    for e, n in enumerate(lengths):
        out.append((e, at, n, fn(e, *(t[at:at + n] for t in tensors)) if n else None))
        at += n
    return out


GROUPS = [([1], 0, 0), ([5, 0, 3], 0, 0), ([0, 0, 17, 0], 2, 5), ([64, 65, 63, 16, 15, 1, 0, 48], 0, 0), ([128, 129, 127, 256, 257], 3, 1), ([300] * 4, 0, 0),
          ([1] * 40, 0, 3), ([0, 700, 0, 0, 90, 2], 0, 0), ([0, 0], 0, 9), ([3] * 256, 1, 1), ([1000, 1, 33], 0, 100)]
SIZES = [(8, 8), (64, 64), (136, 72), (256, 520), (1000, 264), (2056, 1032)]


def product_inputs(lengths, before, after, n, k, seed=51):
    rows = before + sum(lengths) + after
    x = randn(rows, k, seed=seed, dtype=BF16)
    w = randn(len(lengths), n, k, seed=seed + 1, dtype=BF16, scale=k ** -0.5)
    b = randn(len(lengths), n, seed=seed + 2, dtype=BF16)
    dy = randn(rows, n, seed=seed + 3, dtype=BF16)
    for t in (x, dy):           # nobody's rows hold what must not spread
        t[:before] = math.nan
        t[before + sum(lengths):] = math.inf
    return x, w, b, dy


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("lengths,before,after", GROUPS, ids=[f"{len(g[0])}experts{sum(g[0])}rows" for g in GROUPS])
@pytest.mark.parametrize("n,k", SIZES)
def test_grouped_linear(ex, lengths, before, after, n, k, bias):
    if len(lengths) * n * k > 50_000_000:
        pytest.skip("weights of many experts at a small size cover this")
    x, w, b, dy = product_inputs(lengths, before, after, n, k)
    offsets, _ = offsets_of(lengths, before)
    rows = x.shape[0]
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)] + ([b.clone().requires_grad_(True)] if bias else [])
    y = ex.grouped_linear(leaves[0], leaves[1], offsets, leaves[2] if bias else None)
    assert torch.equal(y.detach(), ex.grouped_linear(x, w, offsets, b if bias else None))
    grads = torch.autograd.grad(y, leaves, dy)
    wd, own = w.double(), torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e, at, count, _ in per_expert(lambda e: None, lengths, before):
        if count == 0:
            assert torch.all(grads[1][e] == 0) and (not bias or torch.all(grads[2][e] == 0))
            continue
        own[at:at + count] = True
        xe, we, de = Bound(x[at:at + count].double()), Bound(wd[e]), Bound(dy[at:at + count].double())
        p = matmul(xe, Bound(we.value.t()))
        if bias:
            p = Bound(p.value + b[e].double(), p.err + 2 ** -24 * (p.value.abs() + b[e].double().abs()))
        p.rounded().check(y[at:at + count].detach())
        matmul(de, we).rounded().check(grads[0][at:at + count])
        matmul(Bound(de.value.t()), xe).rounded().check(grads[1][e])
        if bias:
            Bound(de.value.sum(0), (count + 8) * 2 ** -24 * de.value.abs().sum(0)).rounded().check(grads[2][e])
    assert torch.all(y[~own] == 0) and torch.all(grads[0][~own] == 0)


TILES = [(256, 1), (256, -1), (128, -1)]


@pytest.fixture
def tile(request, ex, monkeypatch):
    """Every product on tiles of one kind."""
    import functools

    from bamboo_b200 import lib
    monkeypatch.setattr(lib, "grouped_gemm", functools.partial(lib.grouped_gemm, tile_n=request.param[0], cta_pair=request.param[1]))


@pytest.mark.parametrize("tile", TILES, indirect=True)
@pytest.mark.parametrize("lengths,before,after", GROUPS, ids=[f"{len(g[0])}experts{sum(g[0])}rows" for g in GROUPS])
@pytest.mark.parametrize("n,k", [(64, 64), (136, 72), (520, 1000)])
def test_grouped_linear_on_every_kind_of_tile(ex, tile, lengths, before, after, n, k):
    test_grouped_linear(ex, lengths, before, after, n, k, True)


@pytest.mark.parametrize("rows,experts,n", [(1, 1, 8), (700, 3, 136), (5000, 1, 264), (3000, 40, 1032), (9, 4, 4096)])
def test_a_bias_that_is_trained_alone(ex, rows, experts, n):
    cuts = sorted(torch.randint(0, rows + 1, (experts - 1,), generator=torch.Generator().manual_seed(rows)).tolist())
    at = [0] + cuts + [rows]
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    x, w = randn(rows, 64, seed=1, dtype=BF16), randn(experts, n, 64, seed=2, dtype=BF16)
    bias, dy = randn(experts, n, seed=3, dtype=BF16).requires_grad_(True), randn(rows, n, seed=4, dtype=BF16)
    y = ex.grouped_linear(x, w, offsets, bias)
    (got,) = torch.autograd.grad(y, bias, dy, retain_graph=True)
    arena = torch.nn.Parameter(bias.detach())
    arena.main_grad = randn(experts, n, seed=5)
    before = arena.main_grad.clone()
    ex.grouped_linear(x, w, offsets, arena).backward(dy)
    for e, (a, b) in enumerate(zip(at, at[1:])):
        d = dy[a:b].double()
        want = Bound(d.sum(0), (b - a + 24) * 2 ** -24 * d.abs().sum(0))
        want.rounded().check(got[e])
        Bound(want.value + before[e].double(), want.err + 2 ** -23 * (want.value.abs() + before[e].double().abs())).check(arena.main_grad[e])


@pytest.mark.parametrize("tile", TILES, indirect=True)
def test_an_experts_gradient_does_not_see_its_neighbours_values(ex, tile):
    """Infinities and NaN in one expert's rows stay in its results: in the reduction over rows too, where tiles overhang."""
    lengths, n, k = [37, 50, 21, 1, 130], 136, 72
    x, w, b, dy = product_inputs(lengths, 0, 0, n, k)
    offsets, at = offsets_of(lengths)
    x[at[1]:at[2]], dy[at[3]:at[4]] = math.inf, math.nan
    clean_x, clean_dy = x.clone(), dy.clone()
    clean_x[at[1]:at[2]], clean_dy[at[3]:at[4]] = 1.0, 1.0
    results = []
    for a, d in ((x, dy), (clean_x, clean_dy)):
        leaves = [a.clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
        y = ex.grouped_linear(leaves[0], leaves[1], offsets, leaves[2])
        results.append((y.detach(), *torch.autograd.grad(y, leaves, d)))
    got, want = results
    rows = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
    rows[at[1]:at[2]] = rows[at[3]:at[4]] = False
    assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1][rows], want[1][rows])
    for e in (0, 2, 4):
        assert torch.equal(got[2][e], want[2][e]) and torch.equal(got[3][e], want[3][e])
    assert not torch.isfinite(got[2][1]).all() and not torch.isfinite(got[2][3]).any()


def test_gradients_of_arena_parameters_are_added(ex):
    lengths, n, k = [40, 0, 100, 7], 264, 136
    x, w, b, dy = product_inputs(lengths, 0, 3, n, k)
    offsets, _ = offsets_of(lengths)
    weight, bias = torch.nn.Parameter(w), torch.nn.Parameter(b)
    weight.main_grad, bias.main_grad = randn(*w.shape, seed=60), randn(*b.shape, seed=61)
    before = weight.main_grad.clone(), bias.main_grad.clone()
    y = ex.grouped_linear(x, weight, offsets, bias)
    y.backward(dy)
    assert weight.grad is None and bias.grad is None
    for e, at, count, _ in per_expert(lambda e: None, lengths, 0):
        if not count:
            assert torch.equal(weight.main_grad[e], before[0][e]) and torch.equal(bias.main_grad[e], before[1][e])
            continue
        d, xe = dy[at:at + count].double(), x[at:at + count].double()
        p = matmul(Bound(d.t()), Bound(xe))
        Bound(before[0][e].double() + p.value, p.err + 2 ** -23 * (before[0][e].double().abs() + p.value.abs())).check(weight.main_grad[e])
        s = d.sum(0)
        Bound(before[1][e].double() + s, (count + 9) * 2 ** -24 * (d.abs().sum(0) + before[1][e].double().abs())).check(bias.main_grad[e])


def test_grouped_linear_of_other_strides_and_types_of_offsets(ex):
    lengths, n, k = [30, 12, 0, 70], 72, 64
    x, w, b, dy = product_inputs(lengths, 0, 0, n, k)
    offsets, _ = offsets_of(lengths)
    want = ex.grouped_linear(x, w, offsets, b)
    wide = torch.zeros(x.shape[0], 200, dtype=BF16, device="cuda")
    for at in (0, 8, 3):
        wide[:, at:at + k] = x
        assert torch.equal(ex.grouped_linear(wide[:, at:at + k], w, offsets, b), want)
    assert torch.equal(ex.grouped_linear(x.t().contiguous().t(), w, offsets.long(), b), want)
    assert torch.equal(ex.grouped_linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), offsets, b), want)
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ex.grouped_linear(leaf, w, offsets, b), leaf, dy)
    (h,) = torch.autograd.grad(ex.grouped_linear(leaf, w, offsets, b), leaf, dy.t().contiguous().t())
    assert torch.equal(g, h)
    assert ex.grouped_linear(x[:0], w, torch.zeros(5, dtype=torch.int32, device="cuda"), b).shape == (0, n)
    empty = [x[:0].clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    y = ex.grouped_linear(empty[0], empty[1], torch.zeros(5, dtype=torch.int32, device="cuda"), empty[2])
    for g in torch.autograd.grad(y, empty, dy[:0]):
        assert torch.all(g == 0)


def test_offsets_that_do_not_ascend_are_cut(ex):
    from bamboo_b200 import lib
    x, w, b, _ = product_inputs([40, 30, 30], 0, 0, 64, 64)
    y = ex.grouped_linear(x, w, torch.tensor([0, 70, 40, 1000], dtype=torch.int32, device="cuda"), b)
    torch.cuda.synchronize()
    assert lib.read_status() == -1
    assert torch.equal(y, ex.grouped_linear(x, w, torch.tensor([0, 70, 70, 100], dtype=torch.int32, device="cuda"), b))
    assert lib.read_status() == 0


def gelu(x):
    return torch.nn.functional.gelu(x, approximate="tanh")


def gelu_bound(pre):
    """GeLU of a bound: slope at most 1.13; tanh.approx is off by 2^-10.9 of 1, times half the argument."""
    return Bound(gelu(pre.value), 1.13 * pre.err + 2 ** -11 * (pre.value.abs() + pre.err))


@pytest.mark.parametrize("tile", TILES, indirect=True)
def test_many_tiles_a_cta_on_every_kind(ex, tile):
    """More tiles than CTAs: stages, accumulators and the hand-over of cleaned stages go round many times."""
    test_grouped_linear(ex, [700, 3, 0, 1201, 15, 16, 17, 333, 2, 64, 900, 1], 5, 7, 1544, 776, True)
    test_grouped_linear(ex, [5] * 200, 0, 0, 264, 520, True)


@pytest.mark.parametrize("parts", [2, 3, 7, 32])
@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("lengths,before,after", [([1], 0, 0), ([0, 0], 0, 9), ([64, 65, 0, 127, 1], 3, 1), ([1300, 30], 0, 20)])
@pytest.mark.parametrize("n,k", [(8, 8), (136, 264), (520, 1000)])
def test_weight_gradients_in_parts(ex, lengths, before, after, n, k, tile, parts):
    from bamboo_b200 import lib
    x, _, _, dy = product_inputs(lengths, before, after, n, k, seed=91)
    offsets, _ = offsets_of(lengths, before)
    e, tiles = len(lengths), -(-k // tile[0])
    scratch = torch.full((4 * parts * e * n * (k + tiles),), 255, dtype=torch.uint8, device="cuda")           # (all NaN)
    dw, db = torch.full((e, n, k), math.nan, device="cuda", dtype=BF16), torch.full((e, n), math.nan, device="cuda", dtype=BF16)
    kw = dict(tile_n=tile[0], cta_pair=tile[1], split=parts, bias_parts=scratch)
    lib.grouped_gemm(lib.GROUPED_WEIGHT, dy, x, offsets, dw, bias_grad=db, **kw)
    added, added_b = randn(e, n, k, seed=93), randn(e, n, seed=94)
    before_w, before_b = added.clone(), added_b.clone()
    lib.grouped_gemm(lib.GROUPED_WEIGHT, dy, x, offsets, added, epilogue=lib.EPI_ACCUM_F32, bias_accum=added_b, **kw)
    alone = torch.empty_like(dw)
    lib.grouped_gemm(lib.GROUPED_WEIGHT, dy, x, offsets, alone, **kw)
    assert torch.equal(alone, dw)
    with pytest.raises(lib.BambooNativeError, match="scratch"):
        lib.grouped_gemm(lib.GROUPED_WEIGHT, dy, x, offsets, dw, bias_grad=db, **{**kw, "bias_parts": scratch[:-4 * parts * e * n]})
    for i, at, count, _ in per_expert(lambda e: None, lengths, before):
        rows = slice(at, at + count)
        de = dy[rows].double()
        w = matmul(Bound(de.t()), Bound(x[rows].double())) if count else Bound(torch.zeros(n, k, dtype=torch.float64, device="cuda"))
        w = Bound(w.value, w.err + parts * 2 ** -24 * (de.abs().t() @ x[rows].double().abs()))
        w.rounded().check(dw[i])
        Bound(w.value + before_w[i].double(), w.err + 2 ** -23 * (w.value.abs() + before_w[i].double().abs())).check(added[i])
        b = Bound(de.sum(0), (count + 8 + parts) * 2 ** -24 * de.abs().sum(0))
        b.rounded().check(db[i])
        Bound(b.value + before_b[i].double(), b.err + 2 ** -23 * (b.value.abs() + before_b[i].double().abs())).check(added_b[i])


def test_long_reductions_for_few_tiles_go_in_parts(ex):
    from bamboo_b200 import lib
    lengths = [9000, 13, 4100]
    assert lib.grouped_weight_scratch(sum(lengths), 3, 136, 264, True) > lib.grouped_bias_scratch(3, 136, 264)
    assert lib.grouped_weight_scratch(100, 3, 136, 264, True) == lib.grouped_bias_scratch(3, 136, 264) and lib.grouped_weight_scratch(100, 3, 136, 264, False) == 0
    test_grouped_linear(ex, lengths, 1, 5, 136, 264, True)
    test_grouped_linear(ex, lengths, 0, 0, 136, 264, False)
    test_expert_mlp(ex, [5000, 0, 700], 0, 3, 264, 136)


SPLITS = [(2, 128), (4, 128), (8, 128), (2, 256), (4, 256), (8, 256)]


@pytest.fixture
def split(request, ex, monkeypatch):
    """Reductions shared by so many CTAs wherever they are long enough."""
    from bamboo_b200 import lib
    ctas, tile_n = request.param
    product, calls = lib.grouped_gemm, []

    def shared(mode, x, w, offsets, out, **kw):
        length = -(-x.shape[1] // 64)
        if mode == lib.GROUPED_WEIGHT or length < ctas or (ctas == 8 and x.shape[0] > 96):
            return product(mode, x, w, offsets, out, **kw)
        calls.append(mode)
        return product(mode, x, w, offsets, out, tile_n=tile_n, cta_pair=-1, split=ctas, **kw)

    monkeypatch.setattr(lib, "grouped_gemm", shared)
    return calls


@pytest.mark.parametrize("split", SPLITS, indirect=True)
@pytest.mark.parametrize("n,k", [(136, 520), (1000, 264), (2056, 1032)])
@pytest.mark.parametrize("lengths,before,after", [([1], 0, 0), ([5, 0, 3], 2, 5), ([33, 0, 31, 32], 0, 0), ([0, 0], 0, 9), ([1] * 40, 0, 3), ([64, 65, 127, 129], 3, 1)])
def test_grouped_linear_with_shared_reductions(ex, split, lengths, before, after, n, k):
    test_grouped_linear(ex, lengths, before, after, n, k, True)
    assert split or before + sum(lengths) + after > 96


@pytest.mark.parametrize("split", SPLITS, indirect=True)
def test_epilogues_of_shared_reductions(ex, split):
    from bamboo_b200 import lib
    lengths, before, after, n, k = [40, 0, 7, 33], 2, 3, 1000, 776
    x, w, b, dy = product_inputs(lengths, before, after, n, k, seed=61)
    offsets, _ = offsets_of(lengths, before)
    pre, act, dx = (torch.full((x.shape[0], c), math.nan, device="cuda", dtype=BF16) for c in (n, n, k))
    aux = randn(x.shape[0], k, seed=65, dtype=BF16)
    lib.grouped_gemm(lib.GROUPED_ROWS, x, w, offsets, act, epilogue=lib.EPI_BIAS_GELU, bias=b, out2=pre)
    lib.grouped_gemm(lib.GROUPED_INPUT, dy, w, offsets, dx, epilogue=lib.EPI_MUL_DGELU, aux=aux)
    assert len(split) == 2
    own = torch.zeros(x.shape[0], dtype=torch.bool, device="cuda")
    for e, at, count, _ in per_expert(lambda e: None, lengths, before):
        if not count:
            continue
        rows = slice(at, at + count)
        own[rows] = True
        p = matmul(Bound(x[rows].double()), Bound(w[e].double().t()))
        p = Bound(p.value + b[e].double(), p.err + 2 ** -23 * (p.value.abs() + b[e].double().abs()))
        p.rounded().check(pre[rows])
        gelu_bound(p).rounded().check(act[rows])
        z = aux[rows].double().requires_grad_(True)
        (slope,) = torch.autograd.grad(gelu(z).sum(), z)
        g = matmul(Bound(dy[rows].double()), Bound(w[e].double()))
        # (the slope's tanh is off by 2^-10.9 in two places, as in the expert MLP's test)
        Bound(g.value * slope, g.err * (slope.abs() + 2 ** -9) + g.value.abs() * 2 ** -9).rounded().check(dx[rows])
    assert torch.all(act[~own] == 0) and torch.all(dx[~own] == 0)


@pytest.mark.parametrize("lengths,before,after", [([3], 0, 0), ([40, 0, 130, 7], 0, 5), ([300, 200], 1, 0), ([16] * 12, 0, 0)])
@pytest.mark.parametrize("inner,k", [(64, 64), (264, 136), (1024, 256)])
def test_expert_mlp(ex, lengths, before, after, inner, k):
    rows, e = before + sum(lengths) + after, len(lengths)
    x = randn(rows, k, seed=71, dtype=BF16)
    w1, b1 = randn(e, inner, k, seed=72, dtype=BF16, scale=k ** -0.5), randn(e, inner, seed=73, dtype=BF16, scale=0.2)
    w2, b2 = randn(e, k, inner, seed=74, dtype=BF16, scale=inner ** -0.5), randn(e, k, seed=75, dtype=BF16, scale=0.2)
    dy = randn(rows, k, seed=76, dtype=BF16)
    offsets, _ = offsets_of(lengths, before)
    x[:before], x[before + sum(lengths):], dy[before + sum(lengths):] = math.nan, math.inf, math.nan
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = ex.expert_mlp(leaves[0], offsets, *leaves[1:])
    assert torch.equal(y.detach(), ex.expert_mlp(x, offsets, w1, b1, w2, b2))
    dx, dw1, db1, dw2, db2 = torch.autograd.grad(y, leaves, dy)
    own = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i, at, count, _ in per_expert(lambda e: None, lengths, before):
        if not count:
            assert all(torch.all(g[i] == 0) for g in (dw1, db1, dw2, db2))
            continue
        own[at:at + count] = True
        xe, de = Bound(x[at:at + count].double()), Bound(dy[at:at + count].double())
        v1, v2 = Bound(w1[i].double()), Bound(w2[i].double())
        pre = matmul(xe, Bound(v1.value.t()))
        pre = Bound(pre.value + b1[i].double(), pre.err + 2 ** -23 * (pre.value.abs() + 1))
        act = gelu_bound(pre).rounded()
        out = matmul(act, Bound(v2.value.t()))
        Bound(out.value + b2[i].double(), out.err + 2 ** -23 * (out.value.abs() + 1)).rounded().check(y[at:at + count].detach())
        matmul(Bound(de.value.t()), act).rounded().check(dw2[i])
        Bound(de.value.sum(0), (count + 8) * 2 ** -24 * de.value.abs().sum(0)).rounded().check(db2[i])
        dact = matmul(de, v2)
        pre = pre.rounded()                                             # (the slope is that of the stored one)
        z = pre.value.clone().requires_grad_(True)
        (slope,) = torch.autograd.grad(gelu(z).sum(), z)
        # the slope's own slope is at most 1.13; its tanh is off by 2^-10.9 in two places, the second times |x| (k0 + 3 k0 k1 x^2) (1 - t^2) <= 2
        serr = 1.13 * pre.err + 2 ** -9
        dpre = Bound(dact.value * slope, dact.err * (slope.abs() + serr) + dact.value.abs() * serr).rounded()
        matmul(dpre, v1).rounded().check(dx[at:at + count])
        matmul(Bound(dpre.value.t(), dpre.err.t()), xe).rounded().check(dw1[i])
        s = dpre.value.abs() + dpre.err
        Bound(dpre.value.sum(0), dpre.err.sum(0) + (count + 8) * 2 ** -24 * s.sum(0)).rounded().check(db1[i])
    assert torch.all(y[~own] == 0) and torch.all(dx[~own] == 0)


# ----------------------------------------------------------------------------------- together
def mixture(ex, x, gate, w1, b1, w2, b2, k, normalize=True):
    r = ex.route(torch.nn.functional.linear(x.float(), gate), k, normalize=normalize)
    y = ex.expert_mlp(ex.dispatch(x, r), r.offsets, w1, b1, w2, b2)
    return ex.combine(y, r, residual=x), r


def mixture_inputs(tokens=150, h=64, inner=128, e=5, seed=81):
    return [randn(tokens, h, seed=seed, dtype=BF16), randn(e, h, seed=seed + 1, scale=h ** -0.5), randn(e, inner, h, seed=seed + 2, dtype=BF16, scale=h ** -0.5),
            randn(e, inner, seed=seed + 3, dtype=BF16, scale=0.1), randn(e, h, inner, seed=seed + 4, dtype=BF16, scale=inner ** -0.5),
            randn(e, h, seed=seed + 5, dtype=BF16, scale=0.1)]


@pytest.mark.parametrize("k,normalize", [(1, False), (2, True), (5, False)])
def test_a_mixture_as_it_is_used(ex, k, normalize):
    """Routing, rows out, both layers, rows back, residual, with the balance term: against dense 64-bit autograd over all experts.

    Relative 2-norms: six roundings to bf16 (half a step each, 2^-8) lie between an input and an output or gradient, 6 x 2^-8 = 0.024."""
    inputs = mixture_inputs()
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    dy = randn(150, 64, seed=90, dtype=BF16)
    y, r = mixture(ex, *leaves, k, normalize)
    grads = torch.autograd.grad((y, r.balance), leaves, (dy, torch.tensor(0.5, device="cuda")))
    exact = [t.double().requires_grad_(True) for t in inputs]
    x, gate, w1, b1, w2, b2 = exact
    logits = x @ gate.t()
    member = torch.zeros(150, 5, dtype=torch.bool, device="cuda").scatter_(1, r.experts.long(), True)
    probs = torch.softmax(logits, 1)
    w = torch.softmax(logits.masked_fill(~member, -math.inf), 1) if normalize else torch.where(member, probs, 0.0)
    each = torch.einsum("tei,ehi->teh", gelu(torch.einsum("th,eih->tei", x, w1) + b1), w2) + b2
    want = (w[:, :, None] * each).sum(1) + x
    balance = 5 * (member.double().sum(0) / (150 * k) * probs.mean(0)).sum()
    near(r.balance.detach(), balance.detach(), 2e-5)
    ref = torch.autograd.grad((want, balance), exact, (dy.double(), torch.tensor(0.5, device="cuda", dtype=torch.float64)))
    for got, wanted in zip((y.detach(), *grads), (want.detach(), *ref)):
        assert (got.double() - wanted).norm() <= 0.024 * wanted.norm()


def test_a_mixture_gives_the_same_bits_every_time(ex):
    inputs, dy = mixture_inputs(700, 128, 264, 9), randn(700, 128, seed=91, dtype=BF16)
    runs = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        y, r = mixture(ex, *leaves, 3)
        runs.append([y.detach(), *torch.autograd.grad((y, r.balance), leaves, (dy, torch.tensor(0.5, device="cuda")))])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_a_captured_mixture_follows_its_inputs(ex):
    """Forward and backward pass in a graph, with rows that go elsewhere at every replay.  (No eager graph over the same leaves lives meanwhile:
    autograd would have their gradients wait for the stream of that graph, which breaks the capture of any function.)"""
    inputs, dy = mixture_inputs(), randn(150, 64, seed=92, dtype=BF16)
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            y, r = mixture(ex, *leaves, 2)
            torch.autograd.grad((y, r.balance), leaves, (dy, torch.tensor(0.5, device="cuda")))
    torch.cuda.current_stream().wait_stream(side)
    del y, r
    up = torch.tensor(0.5, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, r = mixture(ex, *leaves, 2)
        grads = torch.autograd.grad((y, r.balance), leaves, (dy, up))
    for seed in (101, 102, 103):
        fresh = mixture_inputs(seed=seed)
        with torch.no_grad():
            for to, t in zip(leaves, fresh):
                to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone().requires_grad_(True) for t in fresh]
        want, rw = mixture(ex, *again, 2)
        ref = torch.autograd.grad((want, rw.balance), again, (dy, up))
        assert torch.equal(y, want) and torch.equal(r.rows, rw.rows)
        assert all(torch.equal(a, b) for a, b in zip(grads, ref))


def test_two_streams_at_once(ex):
    sets = [mixture_inputs(400, 128, 256, 6, seed=s) for s in (111, 121)]
    want = [mixture(ex, *s, 2)[0] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mixture(ex, *sets[i], 2)[0])
    torch.cuda.synchronize()
    for mine, w in zip(got, want):
        assert all(torch.equal(g, w) for g in mine)


def test_second_derivatives_and_overwritten_inputs_are_refused(ex):
    inputs = mixture_inputs(20)
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    y, _ = mixture(ex, *leaves, 2)
    (g,) = torch.autograd.grad(y.float().square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    x, w = inputs[0].clone(), inputs[2].clone().requires_grad_(True)
    y = ex.grouped_linear(x, w, torch.tensor([0, 4, 8, 12, 16, 20], dtype=torch.int32, device="cuda"))
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_two_captured_graphs_at_once(ex):
    """Nothing is shared between captured calls: replays on two streams beside each other, and beside eager calls that need larger scratch."""
    up = torch.tensor(0.5, device="cuda")
    graphs = []
    for seed in (131, 141):
        leaves = [t.requires_grad_(True) for t in mixture_inputs(600, 128, 256, 7, seed=seed)]
        dy = randn(600, 128, seed=seed + 9, dtype=BF16)

        def step(leaves=leaves, dy=dy):
            y, r = mixture(ex, *leaves, 2)
            return [y.detach(), *torch.autograd.grad((y, r.balance), leaves, (dy, up))]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.clone() for t in step()]
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, want, got, torch.cuda.Stream()))
    big = [t.requires_grad_(True) for t in mixture_inputs(3000, 256, 512, 9, seed=151)]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        y, r = mixture(ex, *big, 3)
        torch.autograd.grad(y, big[2], torch.ones_like(y))
    torch.cuda.synchronize()
    for _, want, got, _ in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_offsets_beyond_32_bits(ex):
    """More than 2^31 values in what is read and written."""
    tokens, k, h = 70_000, 8, 4096
    r = ex.route(randn(tokens, 16, seed=161), k)
    x = randn(tokens, h, seed=162, dtype=BF16)
    xs = ex.dispatch(x, r)
    assert xs.numel() > 2 ** 31
    at = torch.tensor([0, 1, tokens * k // 2, tokens * k - 2, tokens * k - 1], device="cuda")
    assert torch.equal(xs[at], x[r.slots[at].long() // k])
    y = ex.combine(xs, r._replace(weights=torch.full_like(r.weights, 1 / 8)))
    assert torch.equal(y, x)                                             # (eight times an eighth of the same row)
    weights = torch.full_like(r.weights, 0.5).requires_grad_(True)
    leaf = xs.requires_grad_(True)
    dxs, dw = torch.autograd.grad(ex.combine(leaf, r._replace(weights=weights)), (leaf, weights), x)
    assert torch.equal(dxs[at], x[r.slots[at].long() // k] * 0.5)
    near(dw[-1], x[-1].double().square().sum().expand(k), 2 ** -24, (h / 16 + 16) * 2 ** -24 * x[-1].double().square().sum())
    del xs, leaf, dxs, y
    rows, n, kk = 140_000, 16384, 64
    cuts = torch.tensor([0, 60_001, 60_001, 139_990], dtype=torch.int32, device="cuda")
    x, w = randn(rows, kk, seed=163, dtype=BF16), randn(3, n, kk, seed=164, dtype=BF16)
    y = ex.grouped_linear(x, w, cuts)
    for a, e in ((0, 0), (60_000, 0), (60_001, 2), (139_989, 2)):
        matmul(Bound(x[a:a + 1].double()), Bound(w[e].double().t())).rounded().check(y[a:a + 1])
    assert torch.all(y[139_990:] == 0)
    dx, dw, = torch.autograd.grad(ex.grouped_linear(a := x.clone().requires_grad_(True), b := w.clone().requires_grad_(True), cuts), (a, b), y)
    matmul(Bound(y[139_989:139_990].double()), Bound(w[2].double())).rounded().check(dx[139_989:139_990])
    matmul(Bound(y[60_001:139_990, -8:].double().t()), Bound(x[60_001:139_990].double())).rounded().check(dw[2, -8:])
    del y, dx, dw, x, w
    e, n, kk = 256, 4096, 2064                                           # the weights
    cuts = torch.arange(0, 2 * e + 1, 2, dtype=torch.int32, device="cuda")
    x, dy = randn(2 * e, kk, seed=165, dtype=BF16), randn(2 * e, n, seed=166, dtype=BF16)
    w = torch.zeros(e, n, kk, dtype=BF16, device="cuda")
    w[-1] = randn(n, kk, seed=167)
    w.requires_grad_(True)
    assert w.numel() > 2 ** 31
    y = ex.grouped_linear(x, w, cuts)
    matmul(Bound(x[-2:].double()), Bound(w[-1].detach().double().t())).rounded().check(y[-2:].detach())
    (dw,) = torch.autograd.grad(y, w, dy)
    matmul(Bound(dy[-2:].double().t()), Bound(x[-2:].double())).rounded().check(dw[-1])


def test_padding_columns_may_hold_anything(ex):
    for n, cols in ((5, 8), (8, 16), (31, 32), (62, 64), (125, 128), (200, 256), (6, 7)):
        for dtype in (FP32, BF16):
            x = randn(300, cols, seed=n, scale=2.0).to(dtype)
            clean = x.clone()
            clean[:, n:] = 0
            x[:, n:] = math.nan
            x[::2, n:] = math.inf
            results = []
            for t in (clean, x):
                leaf = t.clone().requires_grad_(True)
                r = ex.route(leaf, 3, n)
                (g,) = torch.autograd.grad((r.weights, r.balance), leaf, (torch.ones_like(r.weights), torch.tensor(1.0, device="cuda")))
                results.append([r.weights.detach(), r.experts, r.rows, r.slots, r.offsets, r.balance.detach(), g])
            assert all(torch.equal(a, b) for a, b in zip(*results))


def test_one_token_without_a_dimension_for_tokens(ex):
    inputs = mixture_inputs(1)
    r = ex.route(torch.randn(5, device="cuda"), 2)
    assert r.weights.shape == r.rows.shape == (2,)
    x = inputs[0][0]
    rows = ex.dispatch(x, r)
    y = ex.combine(ex.expert_mlp(rows, r.offsets, *inputs[2:]), r, residual=x)
    many = ex.Routing(r.weights[None], r.experts[None], r.rows[None], r.slots, r.offsets)
    assert torch.equal(rows, ex.dispatch(x[None], many)) and y.shape == (64,)
    assert torch.equal(y[None], ex.combine(ex.expert_mlp(rows, r.offsets, *inputs[2:]), many, residual=x[None]))


def test_gradients_of_what_is_shared(ex):
    """One weight for all experts and one bias for all columns, by expand: their gradients are the sums."""
    lengths, n, k = [40, 0, 100, 7], 64, 72
    x, w, _, dy = product_inputs(lengths, 0, 0, n, k)
    offsets, _ = offsets_of(lengths)
    one, value = w[0].clone().requires_grad_(True), torch.tensor(0.5, device="cuda", dtype=BF16, requires_grad=True)
    y = ex.grouped_linear(x, one.expand(4, n, k), offsets, value.expand(4, n))
    dw, dv = torch.autograd.grad(y, (one, value), dy)
    p = matmul(Bound(x.double()), Bound(one.detach().double().t()))
    Bound(p.value + 0.5, p.err + 2 ** -23 * (p.value.abs() + 1)).rounded().check(y.detach())
    d = dy.double()
    # each expert's gradient is rounded to bf16, then autograd adds four, rounding again at most three times
    parts = [matmul(Bound(a.t()), Bound(b)) for a, b in zip(d.split(lengths), x.double().split(lengths)) if len(a)]
    size = sum(q.value.abs() + q.err for q in parts)
    Bound(sum(q.value for q in parts), sum(q.err for q in parts) + 4 * 2 ** -8 * size).check(dw)
    sums = torch.stack([a.sum(0) for a in d.split(lengths)])
    # (256 rounded values, added with at most as many roundings of the partial sum in bf16 or better)
    assert abs(dv.item() - sums.sum().item()) <= 2 ** -8 * (sums.abs().sum().item() + 256 * sums.cumsum(0).abs().max().item())


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (4,), (1, 2), (3, 4), (2, 4), (0, 2), (1, 3)])
def test_some_gradients_of_the_mlp(ex, wanted):
    """Those that are asked for alone, twice over one graph: the same as among all (a bias's sums without its weight go in another order)."""
    lengths = [40, 0, 130, 7, 64]
    offsets, _ = offsets_of(lengths)
    inputs = [randn(241, 136, seed=1, dtype=BF16), *mixture_inputs(1, 136, 264, 5, seed=170)[2:]]
    dy = randn(241, 136, seed=2, dtype=BF16)
    every = [t.clone().requires_grad_(True) for t in inputs]
    full = torch.autograd.grad(ex.expert_mlp(every[0], offsets, *every[1:]), every, dy)
    some = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(inputs)]
    y = ex.expert_mlp(some[0], offsets, *some[1:])
    leaves = [some[i] for i in wanted]
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    for i, a, b in zip(wanted, first, again):
        assert torch.equal(a, b)
        if i in (2, 4) and i - 1 not in wanted:
            # fp32 sums of up to 130 values in two orders, each rounded to bf16
            near(a, full[i].double(), 2 ** -7, 130 * 2 ** -23 * 130)
        else:
            assert torch.equal(a, full[i]), i

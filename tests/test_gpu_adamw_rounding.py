"""8-bit moments over many steps: codes that are rounded up or down at random keep the averages that AdamW is made of; the nearest codes stand still.

Tolerances.  One step on its own: a code is one of the two neighbours of its value, which a 32-bit step makes to 2^-20, and the mean of N such codes is the
value within six standard deviations (each at most half a code step) and the 2^-16 of a step that the random number resolves.

Many steps: rounding x between codes a step s apart adds at most |x - code| s to its variance.  s is an eighth of the root at most in the normal range.  What moves the
root off its code is its own change, (1 - b) |g^2 - v| / 2 in units of v, and that of the block's scale, relative (1 - b) |G^2 / V - 1| / 2 of the largest value's,
which is taken as 2 (1 - b): the largest among several that are nearly so, with E G^2 / V = 3 instead of 1.  So the expected second moment in 8 bits is at most

    u' = b u + (1 - b) (g^2 + (g^2 + u + 4 u) / 16),

while sqrt(b r^2 + c) is convex in r, so that the mean of the root in 8 bits is at least the exact one, r.  The mean of (root / r - 1)^2 is then at most E u / r^2 - 1, that of
root / r at most sqrt(E u / r^2) (Jensen).  Means are over 4096 values and more, whose sample means are off by 3 % at the most here (six times 0.3 / 64).

With b = 0.999 nearest codes end 3 to 7 times too high where gradients have shrunk, or have grown four-fold beside others; with 0.99 throughout, 1.06 times."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
BLOCK = 256
SAMPLE = 0.03


@pytest.fixture(scope="module")
def optim():
    from bamboo_b200 import lib, optim
    lib.load()
    lib.read_status()
    return optim


@pytest.fixture(autouse=True)
def healthy():
    yield
    from bamboo_b200 import lib
    torch.cuda.synchronize()
    assert lib.read_status() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def values(codes, scales):
    return codes.double() * (scales.double() / 256).repeat_interleave(BLOCK)[:codes.numel()]


def state(n, g, offset=0, dtype=FP32):
    """Parameter, master, moments and scales of one tensor, from a random state on."""
    def place(t):
        buf = torch.zeros(n + offset, dtype=t.dtype, device="cuda")
        buf[offset:] = t
        return buf[offset:]
    p = torch.randn(n, device="cuda", generator=g)
    blocks = -(-n // BLOCK)
    m, v = (torch.randn(n, device="cuda", generator=g).mul(60).clamp(-256, 256) for _ in range(2))
    return dict(params=[place(p.to(dtype))], masters=None if dtype == FP32 else [place(p.to(BF16).float())], exp_avgs=[place(m.to(E4M3))],
                exp_avg_sqs=[place(v.abs().to(E4M3))], scales=[torch.rand(2, blocks, device="cuda", generator=g) + 0.5])


def step(optim, s, grad, **kw):
    return optim.adamw_step_(s["params"], [grad], s["exp_avgs"], s["exp_avg_sqs"], scales=s["scales"], masters=s["masters"], **{"rounding": "stochastic", **kw})


def clone(s):
    return {k: None if v is None else [t.clone() for t in v] for k, v in s.items()}


def equal(a, b):
    return all((x is None) == (y is None) and (x is None or torch.equal(x[0].view(torch.uint8), y[0].view(torch.uint8))) for x, y in zip(a.values(), b.values()))


@pytest.mark.parametrize("n", [1, 255, 256, 1000, 77777])
def test_a_code_is_a_neighbour_and_the_mean_of_many_the_value(optim, n):
    g = gen(n)
    start, grad = state(n, g), torch.randn(n, device="cuda", generator=g) * 0.1
    nearest, wide = clone(start), [values(start["exp_avgs"][0], start["scales"][0][0]), values(start["exp_avg_sqs"][0], start["scales"][0][1])]
    step(optim, nearest, grad, step=1000, rounding="nearest")
    m = 0.9 * wide[0] + 0.1 * grad.double()
    r = (0.999 * wide[1] ** 2 + 0.001 * grad.double() ** 2).sqrt()
    total, rounds = [0.0, 0.0], 600
    for at in range(rounds):
        s = clone(start)
        step(optim, s, grad, step=1000 + at)
        if at == 0:
            # the parameter steps on the unrounded moments
            assert torch.equal(s["params"][0], nearest["params"][0]) and torch.equal(s["scales"][0], nearest["scales"][0])
        for i, name in enumerate(("exp_avgs", "exp_avg_sqs")):
            total[i] = total[i] + values(s[name][0], s["scales"][0][i])
            if at < 3:
                scale = s["scales"][0][i].double().repeat_interleave(BLOCK)[:n]
                want = (m, r)[i] * 256 / scale
                size = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -6))) - 3)       # a step of the codes there
                assert ((s[name][0].double() - want).abs() <= size * (1 + 2 ** -16) + 2 ** -18 * want.abs()).all()
    for i, want in enumerate((m, r)):
        scale = nearest["scales"][0][i].double().repeat_interleave(BLOCK)[:n] / 256
        size = scale * torch.exp2(torch.floor(torch.log2((want.abs() / scale).clamp(min=2.0 ** -6))) - 3)
        off = (total[i] / rounds - want).abs()
        assert (off <= size * (3 / math.sqrt(rounds) + 2 ** -16) + 2 ** -18 * want.abs()).all()
        # and over all values, where they are as good as independent
        assert ((total[i] / rounds - want) / size).mean().abs() <= 3 / math.sqrt(rounds * n) + 2 ** -14


@pytest.mark.parametrize("beta2", [0.999, 0.99])
@pytest.mark.parametrize("factor", [1.0, 0.1, 4.0])
@pytest.mark.parametrize("through", ["call", "object"])
def test_roots_follow_gradients_over_thousands_of_steps(optim, beta2, factor, through):
    """Zero-mean gradients of sizes spread over each block; every second value's become `factor` times as large a fifth of the way."""
    n, steps, g = 2 * 4096, 5000, gen(11)
    sizes = torch.exp(torch.randn(n, device="cuda", generator=g)) * 1e-2
    p = torch.zeros(n, device="cuda", requires_grad=True)
    s = dict(params=[p.detach()], masters=None, exp_avgs=[torch.zeros(n, device="cuda", dtype=E4M3)], exp_avg_sqs=[torch.zeros(n, device="cuda", dtype=E4M3)],
             scales=[torch.zeros(2, n // BLOCK, device="cuda")])
    opt = optim.AdamW([p], lr=0.0, betas=(0.9, beta2), state_bits=8)
    v, u = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    for t in range(1, steps + 1):
        if t == steps // 5:
            sizes[::2] *= factor
        grad = sizes * torch.randn(n, device="cuda", generator=g)
        if through == "object":
            p.grad = grad
            opt.step()
        else:
            step(optim, s, grad, step=t, lr=0.0, beta2=beta2)
        sq = grad.double().square()
        v = beta2 * v + (1 - beta2) * sq
        u = beta2 * u + (1 - beta2) * (sq + (sq + 5 * u) / 16)
    codes, scales = (opt.exp_avg_sqs[0], opt.scales[0]) if through == "object" else (s["exp_avg_sqs"][0], s["scales"][0])
    ratio = values(codes, scales[1]) / v.sqrt()
    most = u / v
    for half in (slice(0, None, 2), slice(1, None, 2)):
        assert 1 - SAMPLE <= ratio[half].mean() <= most[half].mean().sqrt() + SAMPLE, ratio[half].mean()
        assert (ratio[half] - 1).square().mean() <= most[half].mean() - 1 + SAMPLE, ratio[half].std()


def test_parameters_move_as_far_as_in_32_bits(optim):
    """A drift that stays while the noise around it shrinks to a tenth: steps that stale roots would hold back.  m / root has the mean of m over r times at least
    1 / E(root / r), and that is at most sqrt(E u / r^2) as above."""
    n, steps, g, beta2 = 2 * 4096, 5000, gen(12), 0.999
    sizes = torch.exp(torch.randn(n, device="cuda", generator=g)) * 1e-2
    params = [torch.zeros(n, device="cuda", requires_grad=True) for _ in range(2)]
    opts = [optim.AdamW([p], lr=1e-3, betas=(0.9, beta2), state_bits=bits) for p, bits in zip(params, (8, 32))]
    u = torch.zeros(n, dtype=torch.float64, device="cuda")
    for t in range(1, steps + 1):
        if t == steps // 5:
            sizes[::2] *= 0.1
            for p in params:
                p.data.zero_()
        grad = sizes * (torch.randn(n, device="cuda", generator=g) + 0.5)
        for p, opt in zip(params, opts):
            p.grad = grad
            opt.step()
        sq = grad.double().square()
        u = beta2 * u + (1 - beta2) * (sq + (sq + 5 * u) / 16)
        if t == steps // 5:
            most = u / opts[1].exp_avg_sqs[0].double()
        else:
            most = u / opts[1].exp_avg_sqs[0].double() if t < steps // 5 else torch.maximum(most, u / opts[1].exp_avg_sqs[0].double())
    for half in (slice(0, None, 2), slice(1, None, 2)):
        moved = [p.detach()[half].double().mean().item() for p in params]
        assert moved[0] / moved[1] >= 1 / math.sqrt(most[half].mean().item()) - SAMPLE


def test_the_same_call_gives_the_same_codes(optim):
    """Wherever tensors begin, whatever stands beside them, captured or not; another step gives others."""
    g = gen(5)
    for dtype in (FP32, BF16):
        grads = [torch.randn(n, device="cuda", generator=g).to(dtype) for n in (1000, 256, 5)]
        both = [[state(n, gen(n), offset=o, dtype=dtype) for n in (1000, 256, 5)] for o in (0, 1, 3)]

        def all_at_once(each, **kw):
            lists = {k: [s[k][0] for s in each] if each[0][k] is not None else None for k in each[0]}
            return optim.adamw_step_(lists["params"], grads, lists["exp_avgs"], lists["exp_avg_sqs"], scales=lists["scales"], masters=lists["masters"],
                                     rounding="stochastic", **kw)
        other = [clone(s) for s in both[0]]
        captured = [clone(s) for s in both[0]]
        for each in both:
            all_at_once(each, step=7, max_norm=1.0)
        assert all(equal(a, b) and equal(a, c) for a, b, c in zip(*both))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            all_at_once(captured, step=7, max_norm=1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(equal(a, b) for a, b in zip(both[0], captured))
        all_at_once(other, step=8, max_norm=1.0)
        assert not torch.equal(other[0]["exp_avgs"][0].view(torch.uint8), both[0][0]["exp_avgs"][0].view(torch.uint8))


def test_tensors_of_one_call_are_rounded_apart(optim):
    """Two alike get codes of their own, in whichever launch they stand; one that is left out leaves the others theirs."""
    n, count = 512, 70
    def make():  # noqa: E306
        each = [state(n, gen(3)) for _ in range(count)]
        return {k: [s[k][0] for s in each] for k in ("params", "exp_avgs", "exp_avg_sqs", "scales")}
    grad = torch.randn(n, device="cuda", generator=gen(4))
    whole, gap = make(), make()
    for lists, grads in ((whole, [grad] * count), (gap, [None] + [grad] * (count - 1))):
        optim.adamw_step_(lists["params"], grads, lists["exp_avgs"], lists["exp_avg_sqs"], scales=lists["scales"], step=3, rounding="stochastic")
    codes = [t.view(torch.uint8) for t in whole["exp_avgs"]]
    assert all(not torch.equal(codes[0], c) for c in codes[1:])
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(codes[1:], gap["exp_avgs"][1:]))


def test_small_and_extreme_values_as_with_nearest_codes(optim):
    n = 4 * BLOCK
    s = dict(params=[torch.zeros(n, device="cuda")], masters=None, exp_avgs=[torch.zeros(n, device="cuda", dtype=E4M3)],
             exp_avg_sqs=[torch.zeros(n, device="cuda", dtype=E4M3)], scales=[torch.zeros(2, 4, device="cuda")])
    g = torch.zeros(n, device="cuda")
    g[0], g[1:BLOCK] = 1.0, 1e-12
    g[BLOCK] = math.inf
    g[2 * BLOCK:2 * BLOCK + 9] = 1e-35
    for at in range(1, 30):
        fresh = clone(s)
        step(optim, fresh, g, step=at)
        scales, m, v = fresh["scales"][0], fresh["exp_avgs"][0].float(), fresh["exp_avg_sqs"][0].float()
        assert m[0] == 256 and v[0] == 256 and torch.all(v[1:BLOCK] == 2 ** -9) and torch.all(m[1:BLOCK] == 0)
        assert scales[:, 0].isfinite().all() and scales[:, 1].isnan().all()
        assert torch.all(m[2 * BLOCK:] == 0) and torch.all(v[3 * BLOCK:] == 0) and torch.all(scales[:, 3] == 0)


def test_saved_states_go_on_alike(optim):
    g = gen(9)
    p = torch.randn(3000, device="cuda", generator=g).to(BF16).requires_grad_(True)
    opt = optim.AdamW([p], lr=1e-2, state_bits=8)
    grads = [torch.randn(3000, device="cuda", generator=g).to(BF16) for _ in range(6)]
    for grad in grads[:3]:
        p.grad = grad
        opt.step()
    q = p.detach().clone().requires_grad_(True)
    other = optim.AdamW([q], state_bits=8)
    other.load_state_dict({k: [t.clone() for t in v] if isinstance(v, list) else v for k, v in opt.state_dict().items()})
    for grad in grads[3:]:
        p.grad, q.grad = grad, grad
        opt.step(), other.step()
    assert torch.equal(p, q) and torch.equal(opt.exp_avg_sqs[0].view(torch.uint8), other.exp_avg_sqs[0].view(torch.uint8))

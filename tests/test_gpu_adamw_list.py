"""The AdamW step over a list of tensors against its formula in 64 bits: types, sizes, alignments, both widths of the moments, clipping, values
out of the ordinary, captured calls.

Tolerances.  A step in 32 bits makes at most eight roundings (2^-24 each) of the terms of every moment, and the update takes about ten more, of
its own size, before it is added to the parameter, one rounding of that: moments 2^-21 of the absolute terms, parameters 2^-23 of themselves plus 2^-19 of
the update.  A working copy is the master rounded to bf16 (2^-8).  8-bit codes: exactly those of the moments that a 32-bit step makes, but where
such a moment, off by 2^-21, lies next to the border of two codes: the code's value is then one step away from the nearest, so it is within half a
step (2^-4 of the value, 2^-10 of the block's top code 256 below the normal range) and 2^-20 more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
BLOCK = 256
ADAM = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)


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


def blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)


def spread(scales, n):
    """[blocks] -> [n]"""
    return scales.repeat_interleave(BLOCK)[:n]


def decode(codes, scales):
    return codes.double().reshape(-1) * (spread(scales.double(), codes.numel()) / 256)


def encode(x):
    """Any valid codes, to start from."""
    b = blocks(x)
    top = b.abs().amax(1)
    code = (b * (256 / top.clamp(min=1e-30))[:, None]).to(E4M3).view(-1)[:x.numel()].clone()
    return code, top


class Lists:
    def __init__(self, sizes, params, grads, bits, seed=1, offset=0):
        g = gen(seed)

        def randn(n, scale):
            return torch.randn(n, device="cuda", generator=g) * scale

        def place(t):
            """The same values ``offset`` elements into a buffer"""
            if not offset:
                return t
            buf = torch.zeros(t.numel() + offset, dtype=t.dtype, device="cuda")
            buf[offset:] = t
            return buf[offset:]
        self.sizes, self.bits = sizes, bits
        start = [randn(n, 0.5) for n in sizes]
        self.masters = [place(p.clone()) for p in start] if params == BF16 else None
        self.params = [place(p.to(params)) for p in start]
        self.grads = [place(randn(n, 0.1).to(gd)) for n, gd in zip(sizes, grads)]
        m, r = [randn(n, 0.05) for n in sizes], [randn(n, 0.1).abs() for n in sizes]
        if bits == 8:
            em, er = [encode(x) for x in m], [encode(x) for x in r]
            self.m, self.v = [place(a) for a, _ in em], [place(a) for a, _ in er]
            self.scales = [torch.stack([a[1], b[1]]) for a, b in zip(em, er)]
        else:
            self.m, self.v, self.scales = [place(x) for x in m], [place(x * x) for x in r], None
        self.before = [self.snapshot(i) for i in range(len(sizes))]

    def snapshot(self, i):
        """(parameter, gradient, first and second moment) in 64 bits"""
        p = (self.masters or self.params)[i].double()
        if self.bits == 8:
            m, v = decode(self.m[i], self.scales[i][0]), decode(self.v[i], self.scales[i][1]).square()
        else:
            m, v = self.m[i].double(), self.v[i].double()
        return p, self.grads[i].double(), m, v

    def step(self, optim, **kw):
        return optim.adamw_step_(self.params, self.grads, self.m, self.v, scales=self.scales, masters=self.masters, **{**ADAM, **kw})


def near(got, want, err):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = torch.isfinite(want)
    over = ((got - want).abs() - err)[ok]
    assert not (over > 0).any(), over.max().item()


def check(lists, coef, step, **kw):
    a = {**ADAM, **kw}
    for i, (p, g, m, v) in enumerate(lists.before):
        g = g * coef
        m1, v1 = a["beta1"] * m + (1 - a["beta1"]) * g, a["beta2"] * v + (1 - a["beta2"]) * g * g
        em, ev = 2 ** -21 * (m.abs() + g.abs()), 2 ** -20 * (v + g * g)
        root = (v1 / (1 - a["beta2"] ** step)).sqrt() + a["eps"]
        update = (m1 / (1 - a["beta1"] ** step)) / root
        e_update = em / (1 - a["beta1"] ** step) / root + 2 ** -19 * update.abs()
        p1 = p - a["lr"] * (update + a["weight_decay"] * p)
        ep = 2 ** -22 * p.abs() + a["lr"] * (e_update + 2 ** -21 * p.abs())
        near((lists.masters or lists.params)[i], p1, ep)
        if lists.masters is not None:
            assert torch.equal(lists.params[i], lists.masters[i].to(BF16))
        if lists.bits == 32:
            near(lists.m[i], m1, em)
            near(lists.v[i], v1, ev)
            continue
        r1 = v1.sqrt()
        for codes, scales, want, e in ((lists.m[i], lists.scales[i][0], m1, em), (lists.v[i], lists.scales[i][1], r1, 2 ** -20 * (v1 + g * g) / r1.clamp(min=1e-30))):
            top = blocks(want).abs().amax(1)
            near(scales, top, blocks(e).amax(1) + 2 ** -22 * top)
            near(decode(codes, scales), want, want.abs() * (2 ** -4 + 2 ** -18) + spread(top, want.numel()) * (2 ** -10 / 256 + 2 ** -20) + 2 * e)


LISTS = [[1], [256], [255, 257, 1, 8], [1000, 4096, 3, 77777], [64] * 70, [7] * 200, [524288 + 5]]


@pytest.mark.parametrize("sizes", LISTS, ids=[f"{len(s)}tensors{sum(s)}" for s in LISTS])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("params,grads", [(FP32, "fp32"), (BF16, "bf16"), (BF16, "mixed")])
def test_a_step(optim, sizes, params, grads, bits):
    types = [FP32 if grads == "fp32" or (grads == "mixed" and i % 2) else BF16 for i in range(len(sizes))]
    for step in (1, 1000):
        lists = Lists(sizes, params, types, bits)
        kept = [g.clone() for g in lists.grads]
        assert lists.step(optim, step=step, grad_scale=0.5) is None
        check(lists, 0.5, step)
        assert all(torch.equal(a, b) for a, b in zip(kept, lists.grads))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("max_norm", [1.0, 1e6])
def test_a_clipped_step(optim, bits, max_norm):
    sizes = [1000, 33, 5000] + [40] * 140
    lists = Lists(sizes, BF16, [BF16] * len(sizes), bits)
    total = torch.cat([g for _, g, _, _ in lists.before]).norm().item() * 0.25
    coef = 0.25 * min(1.0, max_norm / (total + 1e-6))
    norm = lists.step(optim, step=3, grad_scale=0.25, max_norm=max_norm, zero_grad=True)
    assert abs(norm.item() - total) <= 2 ** -22 * total
    check(lists, coef, 3)
    assert all(torch.all(g == 0) for g in lists.grads)
    lists = Lists(sizes, BF16, [BF16] * len(sizes), bits)                  # the norm is over more than this list
    sumsq = torch.tensor([1e4], dtype=torch.float64, device="cuda")
    norm = lists.step(optim, step=3, max_norm=max_norm, sumsq=sumsq)
    assert norm.item() == 100.0
    check(lists, min(1.0, max_norm / (100.0 + 1e-6)), 3)


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_that_start_anywhere(optim, offset, bits):
    lists, plain = (Lists([700, 256, 5], BF16, [BF16, FP32, BF16], bits, offset=o) for o in (offset, 0))
    for l in (lists, plain):
        l.step(optim, step=2, max_norm=1.0)
    for name in ("params", "masters", "m", "v"):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(getattr(lists, name), getattr(plain, name))), name
    if bits == 8:
        assert all(torch.equal(a, b) for a, b in zip(lists.scales, plain.scales))


def test_codes_of_small_and_extreme_values(optim):
    """Roots above 0 keep a code; zeros stay zeros; a block with NaN or infinity is NaN and leaves its neighbours alone."""
    n = 4 * BLOCK
    lists = Lists([n], FP32, [FP32], 8)
    for t in (lists.m[0], lists.v[0]):
        t.view(torch.uint8).zero_()
    lists.scales[0].zero_()
    g = lists.grads[0].zero_()
    g[0], g[1:BLOCK] = 1.0, 1e-12                   # far below the block's largest
    g[BLOCK] = math.inf
    g[2 * BLOCK:2 * BLOCK + 9] = 1e-35              # scales that hold nothing
    lists.step(optim, step=1)
    s, m, v = lists.scales[0], lists.m[0].float(), lists.v[0].float()
    assert s[:, 0].isfinite().all() and m[0] == 256 and v[0] == 256 and torch.all(v[1:BLOCK] == 2 ** -9) and torch.all(m[1:BLOCK] == 0)
    assert s[:, 1].isnan().all()
    assert torch.all(m[2 * BLOCK:] == 0) and torch.all(v[3 * BLOCK:] == 0) and torch.all(s[:, 3] == 0)
    p = lists.params[0]
    assert not torch.isfinite(p[BLOCK]) and torch.isfinite(p[BLOCK + 1:]).all() and torch.isfinite(p[:BLOCK]).all()
    g.zero_()
    lists.step(optim, step=2)
    assert p[BLOCK:2 * BLOCK].isnan().all() and torch.isfinite(p[2 * BLOCK:]).all() and torch.isfinite(p[:BLOCK]).all()


def test_eight_bits_follow_thirty_two(optim):
    """Forty steps on one gradient direction with noise: the parameters of both end near each other (a denominator is off by at most 2^-4, so is a
    first moment: updates by at most 2^-3 + 2^-7 of their size, so are their sums)."""
    n, g = 5000, gen(7)
    ends = []
    for bits in (8, 32):
        p = torch.zeros(n, device="cuda", requires_grad=True)
        opt = optim.AdamW([p], lr=1e-3, betas=(0.9, 0.99), state_bits=bits)
        g = gen(7)
        drift = torch.randn(n, device="cuda", generator=g)
        for _ in range(40):
            p.grad = drift + 0.3 * torch.randn(n, device="cuda", generator=g)
            opt.step()
        ends.append(p.detach())
    assert (ends[0] - ends[1]).norm() <= (2 ** -3 + 2 ** -7) * 40 * 1e-3 * math.sqrt(n)


def test_optimizer_object(optim):
    gens = gen(8)
    params = [torch.randn(s, device="cuda", generator=gens).to(BF16).requires_grad_(True) for s in ((64, 40), (40,), (3, 5, 7))]
    frozen = torch.randn(9, device="cuda").to(BF16)
    opt = optim.AdamW(params + [frozen], lr=1e-2, weight_decay=0.1, state_bits=8, max_norm=1.0)
    params[1].main_grad = torch.randn(40, device="cuda")
    for p in (params[0], params[2]):
        p.grad = torch.randn(p.shape, device="cuda").to(BF16)
    norm = opt.step()
    want = torch.cat([(getattr(p, "main_grad", None) if p.grad is None else p.grad).double().reshape(-1) for p in params]).norm()
    assert abs(norm.item() - want.item()) <= 2 ** -22 * want.item() and opt.step_count == 1
    assert all(torch.equal(p.detach(), m.to(BF16)) for p, m in zip(params, opt.masters))
    assert torch.equal(frozen, opt.params[3])
    other = optim.AdamW([p.detach().clone().requires_grad_(True) for p in params] + [frozen.clone()], state_bits=8)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(opt.params[:3], other.params):
        q.grad = p.grad
        if p.grad is None:
            q.main_grad = p.main_grad.clone()
    opt.step(), other.step()
    assert all(torch.equal(a, b) for a, b in zip(opt.params, other.params))
    opt.zero_grad()
    assert params[0].grad is None and torch.all(params[1].main_grad == 0)
    params[0].grad = None
    assert opt.step().item() == 0.0          # (main_grad zeros alone)


def test_a_parameter_that_was_stepped_is_known_to_autograd(optim):
    p = torch.ones(4, device="cuda", requires_grad=True)
    y = (p * p).sum()
    optim.adamw_step_([p.detach()], [torch.ones(4, device="cuda")], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_captured_step_replays(optim):
    lists, eager = (Lists([3000, 17], BF16, [BF16, BF16], 8) for _ in range(2))
    lists.step(optim, step=5, max_norm=1.0)                        # (buffers that calls keep)
    lists = Lists([3000, 17], BF16, [BF16, BF16], 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = lists.step(optim, step=5, max_norm=1.0)
    for _ in range(3):
        graph.replay()
        want = eager.step(optim, step=5, max_norm=1.0)
        torch.cuda.synchronize()
        assert norm.item() == want.item()
        for name in ("params", "masters", "m", "v", "scales"):
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(getattr(lists, name), getattr(eager, name))), name
    with pytest.raises(Exception, match="cannot be captured"):
        p = torch.zeros(8, device="cuda", requires_grad=True)
        opt, other = optim.AdamW([p]), torch.cuda.CUDAGraph()
        p.grad = torch.ones(8, device="cuda")
        with torch.cuda.graph(other):
            opt.step()


def test_a_tensor_of_more_than_32_bits(optim):
    n = 2 ** 31 + 1000
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda", dtype=BF16)
    m, v = (torch.zeros(n, device="cuda", dtype=E4M3) for _ in range(2))
    s = torch.zeros(2, -(-n // BLOCK), device="cuda")
    ends = torch.tensor([0, 255, 2 ** 31 - 1, 2 ** 31, n - 1], device="cuda")
    g[ends] = 1.0
    optim.adamw_step_([p], [g], [m], [v], scales=[s], step=1, lr=0.5)
    near(p[ends], torch.full((5,), -0.5, device="cuda", dtype=torch.float64), 2 ** -19)
    assert torch.all(m[ends].float() == 256) and torch.all(v[ends].float() == 256)
    assert torch.count_nonzero(p) == 5 and torch.count_nonzero(s) == 2 * 4


def test_two_captured_clipped_steps_at_once(optim):
    sets = [Lists([300_000, 17, 5000], BF16, [BF16] * 3, 8, seed=s) for s in (21, 22)]
    eager = [Lists([300_000, 17, 5000], BF16, [BF16] * 3, 8, seed=s) for s in (21, 22)]
    graphs = []
    for l in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = l.step(optim, step=5, max_norm=0.5)
        graphs.append((graph, norm, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, norm, _), l, e in zip(graphs, sets, eager):
        for _ in range(4):
            want = e.step(optim, step=5, max_norm=0.5)
        assert norm.item() == want.item()
        assert all(torch.equal(a, b) for a, b in zip(l.masters, e.masters))


@pytest.mark.parametrize("bits", [8, 32])
def test_large_and_small_gradients(optim, bits):
    """Second moments as far as 32 bits hold (1 - beta2) g^2: gradients up to 1e20 with beta2 = 0.999, and down to where the square is lost."""
    g = torch.tensor([1e20, -1e20, 1.0, 1e-15, 1e-18], device="cuda")
    for value in g:
        p, m, v = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
        scales = None
        if bits == 8:
            m, v, scales = m.to(E4M3), v.to(E4M3), [torch.zeros(2, 2, device="cuda")]
        optim.adamw_step_([p], [value.expand(300).contiguous()], [m], [v], scales=scales, step=1, lr=1.0, beta2=0.999, eps=0.0)
        # (the first step is the sign of the gradient: m / bias and sqrt(v / bias) are both the gradient's size)
        near(p, -torch.sign(value).double().expand(300), 2 ** -12 if abs(value) < 1e-17 else 2 ** -19)


def test_the_norm_of_a_list_without_gradients_is_on_the_device(optim):
    p = torch.zeros(300, device="cuda", requires_grad=True)
    for opt in (optim.AdamW([p], max_norm=1.0), optim.AdamW([p], max_norm=1.0, state_bits=8)):
        norm = opt.step()
        assert norm.is_cuda and norm.dtype == FP32 and norm.shape == () and norm.item() == 0.0
    assert optim.adamw_step_([], [], [], [], step=1, max_norm=1.0).is_cuda
    assert optim.adamw_step_([p[:0].detach()], [p[:0].detach()], [p[:0].detach()], [p[:0].detach()], step=1, max_norm=1.0).is_cuda

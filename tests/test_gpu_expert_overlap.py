"""A mixture-of-experts half block as redundant work beside the main stream: launched plainly, on a budget, with the same results.

Tolerance: a budget may choose other tiles, whose sums are in another order (2^-24 of their terms); the few results that lie next to the border of two bf16
values then differ by one step (2^-7 of the value), in the second layer too.  2^-8 of the 2-norm is what it would be if half of all did."""
import pytest
import torch

from test_gpu_overlap import _arena, _programmatic_edges

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def restore_budget():
    from bamboo_b200 import lib
    lib.load()
    lib.read_status()
    yield
    lib.GEMM_MAX_CTAS = 0
    torch.cuda.synchronize()
    assert lib.read_status() == 0


@pytest.mark.parametrize("tokens", [(2, 100), (3, 700)])
@pytest.mark.parametrize("budget,overlaps", [(0, True), (-1, False), (20, False)])
def test_experts_beside_the_main_stream_are_launched_plainly(tokens, budget, overlaps):
    from bamboo_b200 import layers, lib
    m = layers.ExpertMLPHalf(256, 6, 512, k=2, seed=2)
    _arena([m])
    x = torch.randn(*tokens, 256, device="cuda").bfloat16()

    def fn():
        with torch.no_grad():
            m(x)
    lib.GEMM_MAX_CTAS = budget
    edges = _programmatic_edges(fn)
    assert edges > 0 if overlaps else edges == 0


@pytest.mark.parametrize("tokens", [1, 130, 2100, 9001])
def test_routing_on_a_budget_gives_the_same_order(tokens):
    from bamboo_b200 import experts as ex
    from bamboo_b200 import lib
    g = torch.Generator(device="cuda").manual_seed(tokens)
    logits = torch.randn(tokens, 40, device="cuda", generator=g).requires_grad_(True)
    dw = torch.randn(tokens, 3, device="cuda", generator=g)
    want = None
    for budget in (0, -1, 1, 20, 1000):
        lib.GEMM_MAX_CTAS = budget
        r = ex.route(logits, 3, 37)
        (grad,) = torch.autograd.grad((r.weights, r.balance), logits, (dw, torch.ones((), device="cuda")))
        if want is None:
            want = r, grad
        for name in ("weights", "experts", "rows", "slots", "offsets"):
            assert torch.equal(getattr(r, name), getattr(want[0], name)), (budget, name)
        # (probabilities are summed by other blocks: 2^-24 of each partial sum, a few hundred at most)
        assert abs(r.balance.item() - want[0].balance.item()) <= 2 ** -16 * want[0].balance.item()
        assert torch.equal(grad, want[1])


@pytest.mark.parametrize("tokens", [(1, 5), (2, 300)])
def test_a_half_block_on_a_budget(tokens):
    from bamboo_b200 import layers, lib
    m = layers.ExpertMLPHalf(256, 6, 512, k=2, seed=2)
    arena = _arena([m])
    g = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.randn(*tokens, 256, device="cuda", generator=g).bfloat16() for _ in range(2))
    want = None
    for budget in (0, -1, 20):
        lib.GEMM_MAX_CTAS = budget
        arena.grad.zero_()
        xi = x.clone().requires_grad_(True)
        y = m(xi)
        y.backward(dy)
        layers.wgrad_sync(x.device)
        got = y.detach().float(), xi.grad.float(), arena.grad.clone()
        want = want or got
        for a, b in zip(got, want):
            assert (a - b).norm() <= 2 ** -8 * b.norm()

"""The global norm of gradients that have run away: values whose squares are no 32-bit numbers any more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pt():
    from bamboo_b200 import lib, post_training
    lib.load()
    lib.read_status()
    return post_training


def lists(dtype, value):
    gen = torch.Generator(device="cuda").manual_seed(71)
    sizes = (1, 7, 4099, 300000)
    grads = [torch.randn(n, device="cuda", generator=gen).to(dtype) for n in sizes]
    yield [g * value for g in grads]                                     # all of them
    grads[2][4098] = value                                               # one behind the last whole vector
    grads[3][12345] = -value                                             # one inside
    yield grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [1e18, 3e19, 1e25, 1e35])
def test_norm_and_clipping_of_large_values(pt, dtype, value):
    """The norm is a 64-bit sum rounded once (2^-24, and 2^-22 for a chunk's squares); what is clipped is scaled by max_norm over it (three roundings, 2^-8
    in bf16)."""
    for grads in lists(dtype, value):
        want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        assert pt.global_grad_norm(grads).item() == pytest.approx(want, rel=5e-7)
        scaled = [g.double() * (1.5 / (want + 1e-6)) for g in grads]
        assert pt.clip_grad_norm_(grads, 1.5).item() == pytest.approx(want, rel=5e-7)
        for g, w in zip(grads, scaled):
            assert ((g.double() - w).abs() <= (2 ** -8 if dtype == torch.bfloat16 else 1e-6) * w.abs() + 1e-38).all()


def test_adam_step_on_large_gradients(pt):
    gen = torch.Generator(device="cuda").manual_seed(72)
    p, g = torch.randn(40000, device="cuda", generator=gen), torch.randn(40000, device="cuda", generator=gen) * 1e22
    want = float(g.double().norm())
    clipped = (g.double() * (0.5 / want)).float()
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    norm = pt.adam_step_clipped(p, g, m, v, None, max_norm=0.5, lr=1e-3, step=1)
    assert norm.item() == pytest.approx(want, rel=5e-7)
    assert torch.allclose(m, 0.1 * clipped, rtol=1e-5, atol=0) and torch.allclose(v, 0.001 * clipped * clipped, rtol=1e-5, atol=0)


def test_infinities_and_nan_stay_what_they_are(pt):
    for bad, norm in ((math.inf, math.inf), (-math.inf, math.inf), (math.nan, math.nan)):
        g = torch.ones(5000, device="cuda")
        g[4321] = bad
        got = pt.global_grad_norm([g]).item()
        assert got == norm or (math.isnan(norm) and math.isnan(got))

"""The router of a mixture-of-experts half block by itself: the gradient of its weight, and of what it reads, with the balance term alone and with the weights of
the chosen rows alone, each held against its own size.

Tolerance: relative 2-norms.  Between input and gradient lie the rounding of the LayerNorm's output, that of the logits' gradient and (weights alone) those of the
activation, the two layers' outputs and the incoming gradient of a row, at most six, half a step of bf16 (2^-8) each: 0.0234.  The output's rounding moves logits by
2^-8 of |h| |gate row| / sqrt(3 hidden) in the mean, below 2^-8 of 2 here, and probabilities by as much of themselves: one more such rounding for a gradient that is linear in them, and
another for the mean that is taken off.  In all 8 x 2^-8 = 0.031."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def healthy():
    from bamboo_b200 import lib
    lib.load()
    lib.read_status()
    yield
    torch.cuda.synchronize()
    assert lib.read_status() == 0


def layer_of(h, experts, k, normalize, coef):
    from bamboo_b200 import layers
    from bamboo_b200.arena import ParamArena
    layer = layers.ExpertMLPHalf(h, experts, 136, k=k, seed=3, balance_coef=coef, normalize=normalize).cuda()
    with torch.no_grad():
        for p in layer.parameters():
            p.add_(torch.randn(p.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(p.numel())) * 0.05)
        layer.gate[:experts].mul_(4.0)
        layer.gate[experts:].zero_()
    ParamArena(layer.parameters(), "cuda")
    return layer


def exact(layer, x, dy, coef):
    """(gradient of the input, {parameter: gradient}) in 64 bits, for the layer's own choice of experts."""
    from bamboo_b200 import experts as E
    from bamboo_b200 import layers
    h, experts, k = x.shape[-1], layer.experts, layer.k
    chosen = E.route(layers._RouterFn.apply(layer.ln(x.detach()), layer, layer.gate.detach()), k, experts, normalize=layer.normalize).experts.view(-1, k)
    P = {n: p.detach().double().requires_grad_(True) for n, p in layer.named_parameters()}
    xd = x.detach().double().view(-1, h).requires_grad_(True)
    hd = torch.nn.functional.layer_norm(xd, (h,), P["ln.weight"], P["ln.bias"], layer.ln.eps)
    logits = hd @ P["gate"][:experts].t()
    member = torch.zeros(len(xd), experts, dtype=torch.bool, device="cuda").scatter_(1, chosen.long(), True)
    probs = torch.softmax(logits, 1)
    w = torch.softmax(logits.masked_fill(~member, -math.inf), 1) if layer.normalize else torch.where(member, probs, 0.0)
    act = torch.nn.functional.gelu(torch.einsum("th,eih->tei", hd, P["fc1_w"]) + P["fc1_b"], approximate="tanh")
    out = (w[:, :, None] * (torch.einsum("tei,ehi->teh", act, P["fc2_w"]) + P["fc2_b"])).sum(1)
    balance = experts * (member.double().sum(0) / (len(xd) * k) * probs.mean(0)).sum()
    ((out * dy.double().view(-1, h)).sum() + coef * balance).backward()
    return xd.grad, {n: p.grad for n, p in P.items()}


def near(got, want):
    assert want.norm() > 0 and (got.double() - want).norm() <= 0.031 * want.norm(), ((got.double() - want).norm() / want.norm()).item()


SHAPES = [(2, 40, 64), (300, 72), (9, 128)]
KINDS = [(5, 2, True), (12, 3, False), (40, 8, True), (7, 1, False)]


@pytest.mark.parametrize("experts,k,normalize", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_the_balance_term_alone(experts, k, normalize, shape):
    layer = layer_of(shape[-1], experts, k, normalize, 0.5)
    layer.balance_grad_scale = 64.0
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(shape, device="cuda", generator=g).bfloat16().requires_grad_(True)
    dy = torch.zeros(shape, device="cuda").bfloat16()
    (dx,) = torch.autograd.grad(layer(x), x, dy)
    want_x, want = exact(layer, x, dy, 0.5 * 64.0)
    torch.cuda.synchronize()
    near(layer.gate.main_grad[:experts], want["gate"][:experts])
    near(dx.view(-1, shape[-1]), want_x)
    assert torch.all(layer.gate.main_grad[experts:] == 0)
    for p in (layer.fc1_w, layer.fc1_b, layer.fc2_w, layer.fc2_b):
        assert torch.all(p.main_grad == 0)


@pytest.mark.parametrize("experts,k,normalize", [kind for kind in KINDS if not kind[2] or kind[1] > 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_the_weights_of_the_rows_alone(experts, k, normalize, shape):
    layer = layer_of(shape[-1], experts, k, normalize, 0.0)
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(shape, device="cuda", generator=g).bfloat16().requires_grad_(True)
    dy = torch.randn(shape, device="cuda", generator=g).bfloat16()
    layer(x).backward(dy)
    _, want = exact(layer, x, dy, 0.0)
    from bamboo_b200 import layers
    layers.wgrad_sync(x.device)
    torch.cuda.synchronize()
    near(layer.gate.main_grad[:experts], want["gate"][:experts])
    assert torch.all(layer.gate.main_grad[experts:] == 0)

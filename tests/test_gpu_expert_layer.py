"""A mixture-of-experts half block as a layer, and a decoder made of them through the pipeline engine.

Tolerances: relative 2-norms.  Between an input and an output or gradient of the layer lie at most eight roundings to bf16 (LayerNorm, activation, the two
layers, the sum, and their counterparts in the backward pass), half a step each: 8 x 2^-8 = 0.031.  In the engine the gradient of a weight is the sum of those of
the micro-batches: the same kernels on the same numbers, added in fp32 (2^-24 each, a few additions whose order is not fixed in dense layers)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def healthy():
    from bamboo_b200 import lib
    lib.load()
    lib.read_status()
    yield
    torch.cuda.synchronize()
    assert lib.read_status() == 0


def gelu(x):
    return torch.nn.functional.gelu(x, approximate="tanh")


@pytest.mark.parametrize("experts,k,normalize", [(1, 1, True), (4, 4, True), (5, 2, True), (12, 3, False)])
@pytest.mark.parametrize("shape", [(2, 40, 64), (1, 1, 128), (300, 72)])
def test_layer_against_dense_64_bit(experts, k, normalize, shape):
    from bamboo_b200 import experts as E
    from bamboo_b200 import layers
    from bamboo_b200.arena import ParamArena
    h, ffn = shape[-1], 136
    layer = layers.ExpertMLPHalf(h, experts, ffn, k=k, seed=3, balance_coef=0.5, normalize=normalize).cuda()
    with torch.no_grad():
        for p in layer.parameters():
            p.add_(torch.randn(p.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(p.numel())) * 0.05)
        layer.gate[:experts].mul_(8.0)                       # far from ties
        layer.gate[experts:].zero_()
    ParamArena(layer.parameters(), "cuda")
    layer.balance_grad_scale = 0.25
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(shape, device="cuda", generator=g).bfloat16().requires_grad_(True)
    dy = torch.randn(shape, device="cuda", generator=g).bfloat16()
    y = layer(x)
    assert torch.equal(y.detach(), layer(x.detach()))
    (dx,) = torch.autograd.grad(y, x, dy)
    # the choice is the layer's own: that of a logit within rounding of another is nobody's fault
    hidden = layer.ln(x.detach())
    chosen = E.route(layers._RouterFn.apply(hidden, layer, layer.gate.detach()), k, experts, normalize=normalize).experts.view(-1, k)
    P = {n: p.detach().double().requires_grad_(True) for n, p in layer.named_parameters()}
    xd = x.detach().double().view(-1, h).requires_grad_(True)
    hd = torch.nn.functional.layer_norm(xd, (h,), P["ln.weight"], P["ln.bias"], layer.ln.eps)
    logits = hd @ P["gate"][:experts].t()
    member = torch.zeros(len(xd), experts, dtype=torch.bool, device="cuda").scatter_(1, chosen.long(), True)
    probs = torch.softmax(logits, 1)
    w = torch.softmax(logits.masked_fill(~member, -math.inf), 1) if normalize else torch.where(member, probs, 0.0)
    each = torch.einsum("tei,ehi->teh", gelu(torch.einsum("th,eih->tei", hd, P["fc1_w"]) + P["fc1_b"]), P["fc2_w"]) + P["fc2_b"]
    want = (w[:, :, None] * each).sum(1) + xd
    balance = experts * (member.double().sum(0) / (len(xd) * k) * probs.mean(0)).sum()
    loss = (want * dy.double().view(-1, h)).sum() + 0.5 * 0.25 * balance
    loss.backward()
    assert abs(layer.balance.item() - balance.item()) <= 2 ** -5 * balance.item()
    pairs = [(y.detach().view(-1, h), want.detach()), (dx.view(-1, h), xd.grad)] + [(p.main_grad, P[n].grad) for n, p in layer.named_parameters()]
    scale = max(P[n].grad.norm().item() for n in ("fc1_w", "fc2_w"))
    for got, ref in pairs:
        # (a gradient that nearly cancels, as the gate's with one expert or all of them, is held against the others' size)
        assert (got.double() - ref).norm() <= 0.031 * ref.norm() + 2 ** -8 * 0.031 * scale, (got.shape, ref.norm().item())


def engine_of(gas, experts=4, layers_=2, lr=1e-3, clipping=0.0):
    from bamboo_b200 import api, models
    from bamboo_b200.module import PipelineModule
    os.environ["BAMBOO_QUIET"] = "1"
    cfg = models.TransformerConfig(layers=layers_, hidden=128, heads=2, ffn=256, seq=64, vocab=500, experts=experts, experts_per_token=2)
    model = PipelineModule(models.transformer_layer_specs(cfg, 0), num_stages=1, loss_fn=models.transformer_loss(cfg), partition_method="uniform")
    engine, *_ = api.initialize(model=model, config={
        "train_micro_batch_size_per_gpu": 4, "gradient_accumulation_steps": gas, "bf16": {"enabled": True}, "gradient_clipping": clipping,
        "optimizer": {"type": "Adam", "params": {"lr": lr}}})
    engine.capture_grads = True
    return engine, cfg


def batches(n, seed=1):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, 500, (n, 4, 65), generator=g)
    return [(t[:, :-1].contiguous(), t[:, 1:].contiguous()) for t in tokens]


def test_a_decoder_with_experts_through_the_engine():
    """The engine's gradients of a step are the sum over its micro-batches, each with the balance terms scaled by 1 / micro-batches."""
    from bamboo_b200 import layers
    gas = 3
    data = batches(gas)
    engine, cfg = engine_of(gas)
    mods = [m for m in engine.module.stages[0].modules.values() if isinstance(m, layers.ExpertMLPHalf)]
    assert len(mods) == 2 and all(m.balance_grad_scale == 1.0 / gas for m in mods)
    loss = engine.train_batch(iter(data))
    got = engine.last_grads[0].clone()
    other, _ = engine_of(gas)
    arena = other.arenas[0]
    arena.grad.zero_()
    total = 0.0
    for tokens, labels in data:
        x = tokens.cuda()
        for m in other.module.stages[0].funcs:
            x = m(x)
        one = other.module.loss_fn(x, labels.cuda()) / gas
        one.backward()
        total += one.item()
    layers.wgrad_sync(torch.device("cuda", torch.cuda.current_device()))
    torch.cuda.synchronize()
    assert abs(float(loss) - total) <= 2 ** -20 * total
    assert (got - arena.grad).norm() <= 2 ** -18 * arena.grad.norm()
    assert all(1.0 <= m.balance.item() < cfg.experts for m in mods)


def test_steps_of_a_decoder_with_experts_and_clipping():
    engine, _ = engine_of(2, experts=6, clipping=0.5)
    data = batches(2, seed=3)
    before = engine.arenas[0].master.clone()
    for _ in range(3):
        loss = engine.train_batch(iter(data))
        assert math.isfinite(float(loss))
    moved = (engine.arenas[0].master - before).abs()
    assert torch.isfinite(engine.arenas[0].master).all() and moved.max() > 0
    assert engine.get_global_grad_norm() > 0

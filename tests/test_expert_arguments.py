"""What the mixture-of-experts and list-optimizer entry points refuse, and what reaches the native calls, as far as that needs no GPU."""
import ctypes

import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture
def recorded(monkeypatch):
    """experts and optim with CPU tensors let through; native calls are recorded instead of made."""
    from bamboo_b200 import experts, lib, optim
    seen = []
    for name in ("grouped_gemm", "grouped_colsum", "expert_mlp_fwd", "expert_mlp_bwd", "route_fwd", "route_bwd", "dispatch_rows", "combine_rows", "combine_rows_bwd",
                 "adamw_list"):
        monkeypatch.setattr(lib, name, lambda *a, _name=name, **kw: seen.append((_name, a, kw)))
    for module in (experts, optim):
        monkeypatch.setattr(module, "_on_current", lambda t, name: None)
    from bamboo_b200 import post_training
    monkeypatch.setattr(post_training, "_on_current", lambda t, name: None)
    return experts, optim, seen


def test_cpu_tensors_are_refused():
    from bamboo_b200 import experts as ex
    from bamboo_b200 import lib, optim
    x, w = torch.zeros(4, 8, dtype=BF16), torch.zeros(2, 8, 8, dtype=BF16)
    offsets, ints = torch.tensor([0, 2, 4]), torch.zeros(4, 1, dtype=torch.int32)
    r = ex.Routing(torch.zeros(4, 1), ints, ints, ints.view(-1), offsets)
    for call in (lambda: ex.route(x, 1), lambda: ex.dispatch(x, r), lambda: ex.combine(x, r), lambda: ex.grouped_linear(x, w, offsets),
                 lambda: ex.expert_mlp(x, offsets, w, w[:, 0], w, w[:, 0]),
                 lambda: optim.adamw_step_([torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], step=1)):
        with pytest.raises(lib.BambooNativeError, match="no CPU fallback"):
            call()


def test_route_refuses(recorded):
    ex, _, seen = recorded
    from bamboo_b200 import lib
    x = torch.zeros(4, 8)
    for k in (0, 9, -1):
        with pytest.raises(ValueError, match="k"):
            ex.route(x, k)
    with pytest.raises(ValueError, match="k 33"):
        ex.route(torch.zeros(4, 64), 33)
    with pytest.raises(ValueError, match="at most 256"):
        ex.route(torch.zeros(4, 257), 2)
    with pytest.raises(ValueError, match="does not fit"):
        ex.route(x, 2, 9)
    with pytest.raises(lib.BambooNativeError, match="bf16 or fp32"):
        ex.route(x.half(), 2)
    assert not seen
    r = ex.route(x.view(2, 2, 8), 2, 5)
    assert r.weights.shape == (2, 2, 2) and r.offsets.shape == (6,) and r.slots.shape == (8,)
    desc = seen[0][1][0]
    assert (desc.tokens, desc.experts, desc.k, desc.normalize, desc.dtype, desc.ld) == (4, 5, 2, 1, 1, 8)


def test_moves_refuse(recorded):
    ex, _, seen = recorded
    from bamboo_b200 import lib
    rows, slots = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    r = ex.Routing(torch.zeros(4, 2), rows, rows, slots, None)
    for bad in (torch.zeros(5, 8), torch.zeros(3, 8)):
        with pytest.raises(ValueError, match="4 tokens"):
            ex.dispatch(bad, r)
    with pytest.raises(lib.BambooNativeError, match="bf16 or fp32"):
        ex.dispatch(torch.zeros(4, 8).half(), r)
    with pytest.raises(ValueError, match="slots"):
        ex.dispatch(torch.zeros(4, 8), r._replace(slots=slots[:7]))
    with pytest.raises(TypeError, match="integers"):
        ex.dispatch(torch.zeros(4, 8), r._replace(rows=rows.float()))
    for bad in (torch.zeros(7, 8), torch.zeros(4, 2, 8)):
        with pytest.raises(ValueError, match="8 places"):
            ex.combine(bad, r)
    with pytest.raises(ValueError, match="weights"):
        ex.combine(torch.zeros(8, 8), r._replace(weights=torch.zeros(4, 3)))
    for bad in (torch.zeros(4, 9), torch.zeros(3, 8), torch.zeros(4, 8, dtype=BF16)):
        with pytest.raises(ValueError, match="residual"):
            ex.combine(torch.zeros(8, 8), r, residual=bad)
    assert not seen


def test_products_refuse(recorded):
    ex, _, seen = recorded
    from bamboo_b200 import lib
    x, w, b, offsets = torch.zeros(6, 16, dtype=BF16), torch.zeros(3, 8, 16, dtype=BF16), torch.zeros(3, 8, dtype=BF16), torch.zeros(4, dtype=torch.int32)
    for bad in (torch.zeros(3, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="one more than there are experts"):
            ex.grouped_linear(x, w, bad, b)
    with pytest.raises(TypeError, match="integers"):
        ex.grouped_linear(x, w, offsets.float(), b)
    for bad in (x.float(), x.half()):
        with pytest.raises(lib.BambooNativeError, match="bf16"):
            ex.grouped_linear(bad, w, offsets, b)
    with pytest.raises(ValueError, match="rows of 16"):
        ex.grouped_linear(x, torch.zeros(3, 8, 24, dtype=BF16), offsets)
    with pytest.raises(ValueError, match="multiples of 8"):
        ex.grouped_linear(x[:, :12], torch.zeros(3, 8, 12, dtype=BF16), offsets)
    with pytest.raises(ValueError, match="multiples of 8"):
        ex.grouped_linear(x, torch.zeros(3, 9, 16, dtype=BF16), offsets)
    with pytest.raises(ValueError, match="1 to 256"):
        ex.grouped_linear(x, torch.zeros(257, 8, 16, dtype=BF16), torch.zeros(258, dtype=torch.int32))
    with pytest.raises(ValueError, match="bias"):
        ex.grouped_linear(x, w, offsets, b[:, :4])
    with pytest.raises(ValueError, match=r"\[rows, values\]"):
        ex.grouped_linear(x.view(2, 3, 16), w, offsets)
    with pytest.raises(ValueError, match=r"\[experts, out, in\]"):
        ex.grouped_linear(x, w[0], offsets)
    with pytest.raises(ValueError, match="both biases"):
        ex.expert_mlp(x, offsets, w, None, torch.zeros(3, 16, 8, dtype=BF16), None)
    with pytest.raises(ValueError, match="one number of experts"):
        ex.expert_mlp(x, offsets, w, b, torch.zeros(2, 16, 8, dtype=BF16), b)
    assert not seen
    ex.grouped_linear(x, w, offsets.long(), b)
    assert seen[0][0] == "grouped_gemm" and seen[0][1][3].dtype == torch.int32


def test_native_calls_refuse_reductions_that_cannot_be_split():
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20
    good = dict(mode=0, rows=64, n=64, k=64, experts=4, epilogue=0, offsets=at, x=at, ld_x=64, weight=at, out=at, ld_out=64)
    for change in (dict(split=3), dict(split=-2), dict(split=16), dict(split=2, max_ctas=8), dict(split=4, tile_n=256, cta_pair=1), dict(split=2, mode=2, ld_weight=64)):
        d = lib.GroupedDesc(**{**good, **change})
        assert handle.bb_grouped_gemm(ctypes.byref(d), None) == -1 and b"split" in handle.bb_last_error(), change


def test_native_calls_refuse_what_python_would_not_send():
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20
    good = dict(mode=0, rows=64, n=64, k=64, experts=4, epilogue=0, offsets=at, x=at, ld_x=64, weight=at, out=at, ld_out=64)
    for change in (dict(rows=0), dict(n=60), dict(k=0), dict(experts=257), dict(offsets=None), dict(offsets=at + 2), dict(mode=3), dict(x=at + 8), dict(ld_x=56), dict(ld_x=68),
                   dict(weight=None), dict(out=None), dict(ld_out=60), dict(epilogue=lib.EPI_BIAS), dict(epilogue=lib.EPI_MUL_DGELU), dict(epilogue=lib.EPI_ACCUM_F32),
                   dict(epilogue=lib.EPI_BIAS_GELU, bias=at), dict(mode=1, epilogue=lib.EPI_BIAS, bias=at), dict(mode=1, epilogue=lib.EPI_MUL_DGELU),
                   dict(mode=2, ld_weight=32), dict(mode=2, ld_weight=64, epilogue=lib.EPI_BIAS, bias=at), dict(tile_n=64), dict(tile_n=96), dict(tile_n=128, cta_pair=1), dict(rows=2 ** 31 - 1), dict(bias_grad=at),
                   dict(mode=2, ld_weight=64, bias_grad=at), dict(mode=2, ld_weight=64, bias_grad=at, bias_parts=at, bias_parts_bytes=64),
                   dict(mode=2, ld_weight=64, bias_grad=at, bias_accum=at, bias_parts=at, bias_parts_bytes=1 << 30)):
        d = lib.GroupedDesc(**{**good, **change})
        assert handle.bb_grouped_gemm(ctypes.byref(d), None) == -1 and b"bb_grouped_gemm" in handle.bb_last_error(), change
    d = lib.GroupedDesc(**{**good, "mode": 2, "ld_weight": 64, "rows": 2 ** 27 + 1})
    assert handle.bb_grouped_gemm(ctypes.byref(d), None) == -4 and b"2^27" in handle.bb_last_error()
    assert handle.bb_grouped_gemm(None, None) == -1 and b"bb_grouped_gemm" in handle.bb_last_error()
    for args in ((None, 64, at, 4, at, None, 8, 64), (at, 64, at, 4, None, None, 8, 64), (at, 64, at, 4, at, at, 8, 64), (at, 64, at, 0, at, None, 8, 64),
                 (at, 64, at, 257, at, None, 8, 64), (at, 64, at, 4, at, None, 0, 64), (at, 64, at, 4, at, None, 8, 60), (at, 32, at, 4, at, None, 8, 64)):
        assert handle.bb_grouped_colsum(*args, None) == -1 and b"bb_grouped_colsum" in handle.bb_last_error(), args
    mlp = dict(rows=8, inputs=64, inner=64, outputs=64, experts=4, offsets=at, w1=at, b1=at, w2=at, b2=at)
    assert handle.bb_expert_mlp_fwd(None, at, 64, at, at, at, None) == -1 and handle.bb_expert_mlp_bwd(None, at, 64, at, at, at, 64, at, at, None) == -1
    for change in (dict(rows=0), dict(inputs=60), dict(inner=0), dict(outputs=12), dict(experts=300), dict(offsets=None), dict(w1=None), dict(b1=None)):
        d = lib.ExpertMLPDesc(**{**mlp, **change})
        assert handle.bb_expert_mlp_fwd(ctypes.byref(d), at, 64, at, at, at, None) == -1, change
    d = lib.ExpertMLPDesc(**mlp)
    assert handle.bb_expert_mlp_fwd(ctypes.byref(d), None, 64, at, at, at, None) == -1
    assert handle.bb_expert_mlp_bwd(ctypes.byref(d), at, 64, at, at, at, 64, None, at, None) == -1 and b"dpre" in handle.bb_last_error()
    d = lib.ExpertMLPDesc(**mlp, dw2=at, db2=at)                                                    # a bias gradient without scratch
    assert handle.bb_expert_mlp_bwd(ctypes.byref(d), at, 64, at, at, at, 64, None, None, None) == -1 and b"bb_grouped_bias_bytes" in handle.bb_last_error()
    route = dict(tokens=16, experts=8, k=2, normalize=1, dtype=0, cols=8, ld=8)
    for change in (dict(tokens=0), dict(experts=0), dict(experts=257), dict(k=0), dict(k=9), dict(experts=64, cols=64, ld=64, k=33), dict(ld=7), dict(cols=7), dict(dtype=2), dict(tokens=1 << 30, k=4)):
        d = lib.RouteDesc(**{**route, **change})
        assert handle.bb_route_workspace_bytes(ctypes.byref(d)) == 0
        assert handle.bb_route_fwd(ctypes.byref(d), *[at] * 10, 1 << 40, None) == -1, change
        assert handle.bb_route_bwd(ctypes.byref(d), *[at] * 7, 512, 256, None) == -1, change
    d = lib.RouteDesc(**route)
    assert handle.bb_route_fwd(ctypes.byref(d), *[at] * 10, 8, None) == -1 and b"workspace" in handle.bb_last_error()
    assert handle.bb_route_bwd(ctypes.byref(d), *[at] * 7, 8, 4, None) == -1
    for args in ((None, 8, 0, at, 2, at, 8, 4, 8), (at, 4, 0, at, 2, at, 8, 4, 8), (at, 8, 2, at, 2, at, 8, 4, 8), (at, 8, 0, at, 0, at, 8, 4, 8), (at, 8, 0, at, 33, at, 8, 4, 8),
                 (at, 8, 0, at, 2, at, 0, 4, 8), (at, 8, 0, at, 2, at, 8, 0, 8), (at + 1, 8, 0, at, 2, at, 8, 4, 8), (at, 8, 0, at, 2, None, 8, 4, 8)):
        assert handle.bb_dispatch_rows(*args, None) == -1 and b"bb_dispatch_rows" in handle.bb_last_error(), args
    assert handle.bb_combine_rows(at, 8, 0, at, at, at, 4, 2, at, 4, 8, 8, None) == -1             # residual rows that overlap
    assert handle.bb_combine_rows_bwd(at, 8, 0, at, 8, at, at, at, 2, None, None, 4, 8, 8, None) == -1       # nothing asked for
    assert handle.bb_combine_rows_bwd(at, 8, 0, at, 8, at, at, at, 2, at, at, 4, 9, 8, None) == -1           # more rows than slots


def lists(n=3, size=300, bits=32, dtype=torch.float32):
    moment = torch.float32 if bits == 32 else torch.float8_e4m3fn
    make = lambda d: [torch.zeros(size, dtype=d) for _ in range(n)]  # noqa: E731
    return dict(params=make(dtype), grads=make(dtype), exp_avgs=make(moment), exp_avg_sqs=make(moment), scales=None if bits == 32 else
                [torch.zeros(2, 2) for _ in range(n)], masters=None if dtype == torch.float32 else make(torch.float32))


def run(optim, args, **kw):
    a = dict(args)
    return optim.adamw_step_(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), **{**a, "step": 1, **kw})


def test_adamw_refuses(recorded):
    _, optim, seen = recorded
    from bamboo_b200 import lib
    for name in ("grads", "exp_avgs", "exp_avg_sqs", "masters"):
        args = lists(dtype=BF16)
        args[name] = args[name][:2]
        with pytest.raises(ValueError, match=name):
            run(optim, args)
        args = lists(dtype=BF16)
        args[name][1] = args[name][1][:299]
        with pytest.raises(ValueError, match=name):
            run(optim, args)
        args = lists(dtype=BF16)
        args[name][1] = args[name][1].half()
        with pytest.raises(lib.BambooNativeError, match=name):
            run(optim, args)
        args = lists(dtype=BF16)
        args[name][1] = torch.zeros(600, dtype=args[name][1].dtype)[::2]
        with pytest.raises(lib.BambooNativeError, match="contiguous"):
            run(optim, args)
    with pytest.raises(lib.BambooNativeError, match="params"):
        run(optim, {**lists(dtype=BF16), "masters": None})             # bf16 parameters without masters
    with pytest.raises(lib.BambooNativeError, match="params"):
        run(optim, {**lists(), "masters": lists()["params"]})
    with pytest.raises(lib.BambooNativeError, match="exp_avgs"):
        run(optim, {**lists(), "scales": lists(bits=8)["scales"]})
    with pytest.raises(ValueError, match="scales"):
        run(optim, {**lists(bits=8), "scales": [torch.zeros(2, 1)] * 3})
    twice = lists()
    twice["params"][2] = twice["params"][0]
    with pytest.raises(ValueError, match="twice"):
        run(optim, twice)
    for kw, what in ((dict(step=0), "step"), (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"), (dict(beta1=1.0), "beta1"),
                     (dict(beta2=-0.1), "beta2")):
        with pytest.raises(ValueError, match=what):
            run(optim, lists(), **kw)
    with pytest.raises(lib.BambooNativeError, match="sumsq"):
        run(optim, lists(), max_norm=1.0, sumsq=torch.zeros(1))
    assert not seen


def test_adamw_leaves_out_what_has_no_gradient(recorded):
    _, optim, seen = recorded
    args = lists(4, bits=8)
    args["grads"][1] = None
    for name in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
        args[name][3] = args[name][3][:0]
    args["scales"][3] = args["scales"][3][:, :0]
    run(optim, args)
    (_, (table, count), _), = seen
    import struct
    fields = struct.unpack("QQQQQQqiI" * count, table)
    assert count == 2 and [fields[0], fields[9]] == [args["params"][0].data_ptr(), args["params"][2].data_ptr()]
    assert [fields[6], fields[15]] == [300, 300] and fields[1] == 0 and fields[5] == args["scales"][0].data_ptr()
    seen.clear()
    args["grads"] = [None] * 4
    assert run(optim, args) is None and run(optim, args, max_norm=1.0) == 0.0 and not seen


def test_adamw_refuses_a_state_that_two_parameters_share(recorded):
    _, optim, seen = recorded
    for kind in (dict(), dict(bits=8), dict(dtype=BF16)):
        for name in ("exp_avgs", "exp_avg_sqs", "scales", "masters"):
            args = lists(**kind)
            if args.get(name) is None:
                continue
            args[name][2] = args[name][0]
            with pytest.raises(ValueError, match="twice"):
                run(optim, args)
        args = lists(**kind)
        args["exp_avg_sqs"] = args["exp_avgs"]
        with pytest.raises(ValueError, match="twice"):
            run(optim, args)
    assert not seen


def test_adamw_without_gradients_still_tells_the_norm_of_all(recorded):
    _, optim, seen = recorded
    args = lists()
    args["grads"] = [None] * len(args["params"])
    norm = run(optim, args, max_norm=1.0, sumsq=torch.full((1,), 9.0, dtype=torch.float64), grad_scale=0.5)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.item() == 1.5 and not seen


def test_optimizer_object_refuses(recorded):
    _, optim, _ = recorded
    from bamboo_b200 import lib
    with pytest.raises(ValueError, match="no parameters"):
        optim.AdamW([])
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([torch.zeros(4)], state_bits=16)
    with pytest.raises(lib.BambooNativeError, match="all fp32 or all bf16"):
        optim.AdamW([torch.zeros(4), torch.zeros(4, dtype=BF16)])
    with pytest.raises(ValueError, match="bits"):
        optim.AdamW([torch.zeros(4)]).load_state_dict(optim.AdamW([torch.zeros(4)], state_bits=8).state_dict())
    with pytest.raises(ValueError, match="not those of these parameters"):
        optim.AdamW([torch.zeros(4)]).load_state_dict(optim.AdamW([torch.zeros(5)]).state_dict())


def test_models_with_experts():
    from bamboo_b200 import layers, models
    cfg = models.TransformerConfig(layers=2, hidden=64, heads=2, ffn=256, seq=32, vocab=100, experts=5, experts_per_token=3)
    names = [s.typename for s in models.transformer_layer_specs(cfg)]
    assert names == [layers.TokenEmbedding, layers.AttentionHalf, layers.ExpertMLPHalf, layers.AttentionHalf, layers.ExpertMLPHalf, layers.LayerNorm, layers.Linear]
    dense = models.TransformerConfig(layers=2, hidden=64, heads=2, ffn=256, seq=32, vocab=100)
    one = models.TransformerConfig(layers=2, hidden=64, heads=2, ffn=256, seq=32, vocab=100, experts=1, experts_per_token=1)
    assert one.flops_per_token() - dense.flops_per_token() == 3 * 2 * 2 * 64
    a, b = (layers.ExpertMLPHalf(64, 5, 256, seed=4) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    assert a.gate.shape == (8, 64) and torch.all(a.gate[5:] == 0)
    with pytest.raises(ValueError, match="3 of 2"):
        layers.ExpertMLPHalf(64, 2, 256, k=3)


def test_layers_learn_the_engines_factor():
    from bamboo_b200 import layers
    from bamboo_b200.module import LayerSpec, PipelineModule
    m = PipelineModule([LayerSpec(layers.ExpertMLPHalf, 16, 2, 32), LayerSpec(torch.nn.Linear, 4, 4)], num_stages=1, loss_fn=None, partition_method="uniform")
    layer = next(iter(m.stages[0].modules.values()))
    assert layer.balance_grad_scale == 1.0
    m.scale_layer_gradients(0.25)
    assert layer.balance_grad_scale == 0.25
    m.build_layers(0)
    assert next(iter(m.stages[0].modules.values())).balance_grad_scale == 0.25


def test_arena_gradients_that_kernels_could_not_add_to(recorded):
    ex, _, _ = recorded
    from bamboo_b200 import lib
    for bad in (torch.zeros(2, 8, 8, dtype=BF16), torch.zeros(2, 8, 9), torch.zeros(2, 8, 16)[..., ::2], torch.zeros(129)[1:].view(2, 8, 8)):
        p = torch.nn.Parameter(torch.zeros(2, 8, 8, dtype=BF16))
        p.main_grad = bad
        with pytest.raises(lib.BambooNativeError, match="main_grad"):
            ex._arena_gradient(p)
    p.main_grad = torch.zeros(2, 8, 8)
    assert ex._arena_gradient(p) is p.main_grad


def test_constants_given_as_tensors(recorded):
    _, optim, seen = recorded
    value = torch.tensor(0.25)
    for want in (0.25, 0.5):
        value.fill_(want)
        run(optim, lists(), lr=value, weight_decay=value, beta1=value, grad_scale=value)
        assert [seen[-1][2][n] for n in ("lr", "weight_decay", "beta1", "grad_scale")] == [want] * 4


def test_native_list_step_refuses():
    import struct
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20

    def call(param=at, master=0, grad=at, m=at, v=at, scales=0, numel=300, dtype=1, count=1, step=1, beta1=0.9, max_norm=0.0, norm=None, ws=None, ws_bytes=0):
        table = struct.pack("QQQQQQqiI", param, master, grad, m, v, scales, numel, dtype, 0)
        return handle.bb_adamw_list(table, count, 1e-3, beta1, 0.999, 1e-8, step, 0.0, 1.0, 0, max_norm, None, norm, ws, ws_bytes, None)
    for bad in (dict(param=0), dict(grad=0), dict(m=0), dict(v=0), dict(numel=0), dict(numel=-1), dict(numel=1 << 39), dict(dtype=2), dict(param=at + 2), dict(param=at + 1, master=at),
                dict(master=at + 2), dict(grad=at + 2), dict(grad=at + 1, dtype=0), dict(m=at + 2), dict(scales=at + 2), dict(count=0), dict(count=-1), dict(step=0), dict(beta1=1.0),
                dict(max_norm=-1.0), dict(max_norm=1.0), dict(max_norm=1.0, norm=at, ws=at, ws_bytes=16), dict(max_norm=1.0, norm=at, ws=at + 4, ws_bytes=1 << 20)):
        assert call(**bad) == -1 and b"bb_adamw_list" in handle.bb_last_error(), bad


def test_rounding_of_codes(recorded):
    _, optim, seen = recorded
    import struct
    for bad in ("up", None, 1):
        with pytest.raises(ValueError, match="rounding"):
            run(optim, lists(bits=8), rounding=bad)
    assert not seen
    for rounding, want in (("nearest", [0, 0]), ("stochastic", [1, 3])):
        args = lists(bits=8)
        args["grads"][1] = None
        run(optim, args, rounding=rounding)
        table, count = seen[-1][1]
        assert list(struct.unpack("QQQQQQqiI" * count, table)[8::9]) == want
    p = torch.zeros(300, requires_grad=True)
    p.grad = torch.ones(300)
    opt = optim.AdamW([p], state_bits=8)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        opt.step()
    assert struct.unpack("QQQQQQqiI", seen[-1][1][0])[8] == 1


def test_native_list_step_refuses_seeds_for_a_part_of_a_list():
    import struct
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20
    table = struct.pack("QQQQQQqiI" * 2, *(at, 0, at, at, at, at, 300, 1, 1), *(at, 0, at, at, at, at, 300, 1, 0))
    assert handle.bb_adamw_list(table, 2, 1e-3, 0.9, 0.999, 1e-8, 1, 0.0, 1.0, 0, 0.0, None, None, None, 0, None) == -1 and b"seeds" in handle.bb_last_error()


def test_native_expert_mlp_refuses_scratch_before_anything_is_launched():
    """Gradients added to an arena would be added twice by a caller that tries again after a refusal half way."""
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20
    mlp = dict(rows=8, inputs=64, inner=64, outputs=64, experts=4, offsets=at, w1=at, b1=at, w2=at, b2=at)
    for layer in (dict(g_w1=at), dict(dw1=at), dict(g_w2=at), dict(dw2=at), dict(g_w1=at, g_w2=at)):
        for scratch in (dict(scratch=at + 8, scratch_bytes=1 << 20), dict(scratch_bytes=64), dict(scratch=at + 4)):
            d = lib.ExpertMLPDesc(**mlp, **layer, **scratch)
            assert handle.bb_expert_mlp_bwd(ctypes.byref(d), at, 64, at, at, at, 64, at, at, None) == -1, (layer, scratch)
            assert b"bb_expert_mlp_bwd" in handle.bb_last_error() and b"scratch" in handle.bb_last_error(), handle.bb_last_error()
    for layer in (dict(db1=at), dict(g_b2=at)):                              # bias gradients alone cover 65535 x 128 columns
        sizes = dict(inner=1 << 23) if "db1" in layer else dict(outputs=1 << 23)
        d = lib.ExpertMLPDesc(**{**mlp, **sizes}, **layer)
        assert handle.bb_expert_mlp_bwd(ctypes.byref(d), at, 64, at, at, at, 1 << 23, at, at, None) == -1
        assert b"bb_expert_mlp_bwd" in handle.bb_last_error() and b"columns" in handle.bb_last_error()


def test_routing_beside_the_main_stream_is_told_its_budget(recorded, monkeypatch):
    ex, _, seen = recorded
    from bamboo_b200 import lib
    for budget in (0, 20, -1, 0):
        monkeypatch.setattr(lib, "GEMM_MAX_CTAS", budget)
        ex.route(torch.zeros(4, 8), 2)
        assert seen[-1][1][0].max_ctas == budget


@pytest.mark.parametrize("kind", [dict(), dict(bits=8), dict(dtype=BF16)])
def test_adamw_refuses_tensors_that_share_memory(recorded, kind):
    """Not only those that begin at one address: a value that two CTAs step on has the last one's result."""
    _, optim, seen = recorded
    for name in ("params", "exp_avgs", "exp_avg_sqs", "scales", "masters"):
        args = lists(**kind)
        if args.get(name) is None:
            continue
        buffer = torch.zeros(900, dtype=args[name][0].dtype)
        shape, n = args[name][0].shape, args[name][0].numel()
        args[name][:2] = [buffer[at:at + n].view(shape) for at in (0, n - 1)]
        with pytest.raises(ValueError, match="shares memory"):
            run(optim, args)
        args[name][:2] = [buffer[at:at + n].view(shape) for at in (n, 0)]                # neighbours
        run(optim, args)
        assert seen.pop()
    args = lists(**kind)
    both = torch.zeros(599, dtype=args["grads"][0].dtype)
    args["grads"][:2] = both[:300], both[299:]
    run(optim, args)                                      # gradients that overlap are only read ...
    assert seen.pop()
    with pytest.raises(ValueError, match="zeroed"):       # ... unless they are zeroed while another reads them
        run(optim, args, zero_grad=True)
    args["grads"][1] = args["grads"][0]
    with pytest.raises(ValueError, match="zeroed"):
        run(optim, args, zero_grad=True)
    args = lists(**kind)
    if "bits" not in kind:
        place = "masters" if kind else "params"
        args["grads"][0] = args[place][2]                 # a gradient that the step overwrites
        with pytest.raises(ValueError, match="shares memory"):
            run(optim, args)
    assert not seen


def test_native_list_tells_of_shared_memory():
    import random
    import struct
    from bamboo_b200 import lib
    handle, rng = lib.load(), random.Random(3)
    assert handle.bb_adamw_list_overlaps(None, 1, 0) == 0
    for _ in range(300):
        count, bits, zero = rng.randint(1, 9), rng.choice([8, 32]), rng.randint(0, 1)
        rows, ranges = [], []
        for _ in range(count):
            n, master, dtype = rng.randint(1, 700), rng.randint(0, 1), rng.randint(0, 1)
            place = lambda size: rng.randrange(16, 1 << rng.choice([15, 22]), 8) if size else 0  # noqa: E731
            sizes = (2 * n if master else 4 * n, 4 * n * master, (2, 4)[dtype] * n, n * bits // 8, n * bits // 8, 8 * -(-n // 256) * (bits == 8))
            at = [place(size) for size in sizes]
            rows += [*at, n, dtype, 0]
            ranges += [(a, a + size, i != 2 or zero) for i, (a, size) in enumerate(zip(at, sizes)) if size]
        want = any(a[0] < b[1] and b[0] < a[1] and (a[2] or b[2]) for i, a in enumerate(ranges) for b in ranges[:i])
        assert handle.bb_adamw_list_overlaps(struct.pack("QQQQQQqiI" * count, *rows), count, zero) == want


def test_rows_that_32_bits_do_not_count(recorded):
    """A size of 2^32 + 8 would reach the native call as 8."""
    ex, _, seen = recorded
    from bamboo_b200 import lib
    wide = torch.zeros(1, 1).expand(4, 2 ** 32 + 8)
    ints = torch.zeros(4, 1, dtype=torch.int32)
    r = ex.Routing(torch.zeros(4, 1), ints, ints, ints.view(-1), None)
    for call in (lambda: ex.dispatch(wide, r), lambda: ex.combine(wide, r), lambda: ex.dispatch(wide[:, :2 ** 31 - 8], r)):
        with pytest.raises(ValueError, match="values, at most"):
            call()
    with pytest.raises(ValueError, match="columns, at most"):
        ex.route(wide, 1, 8)
    many = torch.zeros(1, 1, dtype=torch.int32).expand(2 ** 31, 1)
    with pytest.raises(ValueError, match="rows, at most"):
        ex.dispatch(torch.zeros(1, 1).expand(2 ** 31, 8), r._replace(rows=many, slots=many.view(-1)))
    x, offsets = torch.zeros(6, 8, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    for shape in ((1, 2 ** 32 + 8, 8), (1, 8, 2 ** 32 + 8)):
        with pytest.raises(ValueError, match="sizes of at most"):
            ex.grouped_linear(x, torch.zeros(1, 1, 1, dtype=BF16).expand(shape), offsets)
    assert not seen
    handle, at, n = lib.load(), 1 << 20, 2 ** 31 - 8
    good = dict(mode=0, rows=64, n=64, k=64, experts=4, epilogue=0, offsets=at, x=at, ld_x=64, weight=at, out=at, ld_out=64)
    for change in (dict(n=n, ld_out=n), dict(k=n, ld_x=n), dict(mode=1, k=n, ld_out=n), dict(mode=2, k=n, ld_weight=n)):
        assert handle.bb_grouped_gemm(ctypes.byref(lib.GroupedDesc(**{**good, **change})), None) == -1, change
    mlp = dict(rows=8, inputs=64, inner=64, outputs=64, experts=4, offsets=at, w1=at, b1=at, w2=at, b2=at)
    for name in ("inputs", "inner", "outputs"):
        d = lib.ExpertMLPDesc(**{**mlp, name: n})
        assert handle.bb_expert_mlp_fwd(ctypes.byref(d), at, n, at, at, at, None) == -1
        assert handle.bb_expert_mlp_bwd(ctypes.byref(d), at, n, at, at, at, n, at, at, None) == -1
    d = lib.RouteDesc(tokens=16, experts=8, k=2, normalize=1, dtype=0, cols=n, ld=n)
    assert handle.bb_route_fwd(ctypes.byref(d), *[at] * 10, 1 << 40, None) == -1 and handle.bb_route_bwd(ctypes.byref(d), *[at] * 7, n, 8, None) == -1
    d = lib.RouteDesc(tokens=16, experts=8, k=2, normalize=1, dtype=0, cols=8, ld=8)
    assert handle.bb_route_bwd(ctypes.byref(d), *[at] * 7, n, n, None) == -1
    assert handle.bb_dispatch_rows(at, n, 0, at, 2, at, 8, 4, n, None) == -1
    assert handle.bb_combine_rows(at, n, 0, at, at, None, 0, 2, at, 4, 8, n, None) == -1
    assert handle.bb_combine_rows_bwd(at, n, 0, at, n, at, at, at, 2, at, at, 4, 8, n, None) == -1

"""``gradient_clipping`` on CPU ranks (gloo): the norm is over the whole model wherever its stages live, clipped steps follow a
single-process trainer that clips with torch, through a failover too; and what the post-training entry points refuse without a GPU."""
import ctypes
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from oracle import gpt_ref  # noqa: E402

CFG = gpt_ref.RefConfig(layers=4, hidden=64, heads=4, ffn=128, seq=16, vocab=96)
MB, GAS, STEPS, LR, LIMIT = 2, 4, 4, 1e-3, 0.5


def _train(rank, world, store, stages, rc, limit, victim_step):
    import cpu_layers
    from bamboo_b200 import api
    from bamboo_b200.module import PipelineModule
    model = PipelineModule(cpu_layers.ref_layer_specs(CFG, 0), num_stages=stages, loss_fn=cpu_layers.ref_loss(CFG),
                           partition_method="uniform", device="cpu")
    config = {"train_micro_batch_size_per_gpu": MB, "gradient_accumulation_steps": GAS, "gradient_clipping": limit,
              "optimizer": {"type": "Adam", "params": {"lr": LR}}, "bamboo_b200": {"p2p_timeout_s": 20}}
    engine, *_ = api.initialize(model=model, config=config, redundancy_level=rc, store=store if world > 1 else None)
    engine.capture_grads = True
    losses, norms, grads = [], [], []
    for step, batches in enumerate(gpt_ref.synthetic_batches(CFG, MB, GAS, STEPS, seed=1)):
        if victim_step is not None and step == victim_step - 1 and rank == stages - 1:
            engine.announce_preemption()
        losses.append(float(engine.train_batch(data_iter=iter(batches))))
        norms.append(engine.get_global_grad_norm())
        grads.append(float(sum(g.double().square().sum() for g in engine.last_grads.values())))
    return {"losses": losses, "norms": norms, "sumsq": grads, "stage_ids": list(engine.stage_ids),
            "checksum": {s: float(engine.arenas[s].master.double().sum()) for s in engine.stage_ids},
            "master": engine.arenas[0].master.tolist() if world == 1 else None}


def _single(limit):
    os.environ["BAMBOO_QUIET"] = "1"
    return _train(0, 1, None, 1, 0, limit, None)


def test_single_stage_clips_like_torch():
    """One engine step against torch's clipping and AdamW in 64 bits on the engine's own captured gradients."""
    import cpu_layers
    from bamboo_b200 import api
    from bamboo_b200.module import PipelineModule
    os.environ["BAMBOO_QUIET"] = "1"
    model = PipelineModule(cpu_layers.ref_layer_specs(CFG, 0), num_stages=1, loss_fn=cpu_layers.ref_loss(CFG), partition_method="uniform",
                           device="cpu")
    engine, *_ = api.initialize(model=model, config={"train_micro_batch_size_per_gpu": MB, "gradient_accumulation_steps": GAS,
                                                     "gradient_clipping": LIMIT, "optimizer": {"type": "Adam", "params": {"lr": LR}}})
    engine.capture_grads = True
    assert engine.get_global_grad_norm() is None
    (batches,) = gpt_ref.synthetic_batches(CFG, MB, GAS, 1, seed=1)
    before = engine.arenas[0].master.clone()
    engine.train_batch(data_iter=iter(batches))
    p = torch.nn.Parameter(before.double())
    p.grad = engine.last_grads[0].double()
    norm = torch.nn.utils.clip_grad_norm_([p], LIMIT)
    assert norm > LIMIT and engine.get_global_grad_norm() == pytest.approx(float(norm), rel=1e-6)
    torch.optim.AdamW([p], lr=LR, weight_decay=0.0).step()
    assert torch.allclose(engine.arenas[0].master.double(), p.detach(), rtol=1e-5, atol=1e-8)
    assert torch.all(engine.arenas[0].grad == 0)


def test_a_limit_that_is_not_reached_changes_nothing():
    free, loose = _single(0.0), _single(1e6)
    assert free["norms"] == [None] * STEPS and free["losses"] == loose["losses"]
    assert free["master"] == loose["master"]
    assert loose["norms"] == pytest.approx([math.sqrt(s) for s in loose["sumsq"]], rel=1e-6)


@pytest.mark.parametrize("rc,victim_step", [(0, None), (1, None), (1, 2)])
def test_pipeline_clips_over_all_stages(rc, victim_step):
    from dist_utils import run_ranks
    want = _single(LIMIT)
    assert min(want["norms"]) > LIMIT
    res = run_ranks(_train, 2, 2, rc, LIMIT, victim_step)
    if victim_step is None:
        outs = [res[r][1] for r in range(2)]
        assert [res[r][0] for r in range(2)] == ["ok", "ok"]
        assert outs[0]["norms"] == outs[1]["norms"]
        for step in range(STEPS):
            assert outs[0]["norms"][step] == pytest.approx(math.sqrt(outs[0]["sumsq"][step] + outs[1]["sumsq"][step]), rel=1e-6)
        assert outs[1]["losses"] == pytest.approx(want["losses"], rel=1e-4)
        total = sum(o["checksum"][s] for s, o in enumerate(outs))
    else:
        assert res[1] == ("exit", 13)
        status, out = res[0]
        assert status == "ok" and out["stage_ids"] == [0, 1], out
        outs = [out]
        assert out["losses"][victim_step:] == pytest.approx(want["losses"][victim_step:], rel=1e-4)
        total = sum(out["checksum"].values())
    assert outs[0]["norms"] == pytest.approx(want["norms"], rel=1e-4)
    assert total == pytest.approx(want["checksum"][0], rel=1e-5)


def test_a_stage_that_never_publishes_is_an_error():
    from types import SimpleNamespace
    from bamboo_b200.engine import LocalStore, PipelineEngine, PipelineError
    arena = SimpleNamespace(grad_sumsq=lambda: torch.ones(1, dtype=torch.float64))
    grid = SimpleNamespace(get_data_parallel_id=lambda: 0)
    me = SimpleNamespace(stage_ids=[0], num_stages=2, arenas={0: arena}, _clip_epoch=0, global_steps=3, grid=grid, global_store=LocalStore(),
                         _config=SimpleNamespace(p2p_timeout_s=0.05), device=torch.device("cpu"))
    me.global_store.set("grad-sumsq-0-1-1", "0-1:4.0")                # an earlier step's number is not taken
    with pytest.raises(PipelineError, match="stage 1"):
        PipelineEngine._pipeline_sumsq(me, {0: 0.5})
    me.global_store.set("grad-sumsq-0-1-1", "0-3:4.0")
    assert float(PipelineEngine._pipeline_sumsq(me, {0: 0.5})) == 4.25
    assert me.global_store.get("grad-sumsq-0-0-1") == b"0-3:0.25"


# ----------------------------------------------------------------------------------- argument checks that need no GPU
def test_native_refusals_do_not_need_a_gpu():
    from bamboo_b200 import lib
    handle, at = lib.load(), 1 << 20

    def refused(rc, text):
        assert rc == -1 and text in handle.bb_last_error(), (rc, handle.bb_last_error())
    fwd = lambda **kw: handle.bb_token_logprob_fwd(*{**dict(logits=at, dtype=0, ld=64, targets=at, scale=1.0, logp=at, stats=at, rows=4, vocab=64,  # noqa: E731
                                                            ignore=-100, stream=None), **kw}.values())
    for bad in (dict(logits=None), dict(targets=None), dict(dtype=2), dict(ld=63), dict(rows=0), dict(vocab=0), dict(scale=0.0), dict(scale=math.nan),
                dict(logits=at + 1), dict(logp=None), dict(stats=at + 4)):
        refused(fwd(**bad), b"bb_token_logprob_fwd")
    bwd = lambda **kw: handle.bb_token_logprob_bwd(*{**dict(logits=at, dtype=1, ld=64, targets=at, scale=1.0, stats=at, row_grad=at, dev=None, g=1.0,  # noqa: E731
                                                            d=1 << 30, ldd=64, rows=4, vocab=60, cols=64, ignore=-100, stream=None), **kw}.values())
    for bad in (dict(row_grad=None), dict(cols=59), dict(ldd=63), dict(d=(1 << 30) + 2), dict(d=at, ldd=65, cols=64), dict(d=at + 4)):
        refused(bwd(**bad), b"bb_token_logprob_bwd")
    d = lib.PreferenceDesc(tokens=8, sequences=2, form=0, beta=0.1, label_smoothing=0.0, average=0, ignore_index=-100)

    def preference(ws=1 << 20, **kw):
        e = lib.PreferenceDesc(**{n: kw.get(n, getattr(d, n)) for n, _ in d._fields_})
        return handle.bb_preference_loss(ctypes.byref(e), at, None, at, None, at, at, at, at, ws, None)
    for bad in (dict(tokens=0), dict(sequences=3), dict(sequences=0), dict(tokens=7), dict(form=3), dict(beta=0.0), dict(label_smoothing=2.0), dict(ws=4)):
        refused(preference(**bad), b"bb_preference_loss")
    q = lib.PolicyDesc(tokens=8, sequences=2, reduction=0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, advantage_per_sequence=0, ignore_index=-100)

    def policy(ws=1 << 20, offsets=None, **kw):
        e = lib.PolicyDesc(**{n: kw.get(n, getattr(q, n)) for n, _ in q._fields_})
        return handle.bb_policy_loss(ctypes.byref(e), at, None, at, None, at, offsets, at, at, at, at, ws, None)
    for bad in (dict(tokens=0), dict(sequences=0), dict(tokens=7), dict(reduction=2), dict(clip_low=-1.0), dict(clip_high=math.nan), dict(kl_coef=-1.0),
                dict(ws=8), dict(offsets=at, advantage_per_sequence=1)):
        refused(policy(**bad), b"bb_policy_loss")
    h = dict(rows=4, vocab=100, hidden=64, ld_hidden=64, ld_weight=64, scale=1.0, ignore_index=-100)

    def head(ws=1 << 20, states=at, **kw):
        return handle.bb_head_logprob_fwd(ctypes.byref(lib.HeadDesc(**{**h, **kw})), states, at, at, at, at, at, ws, None)
    for bad in (dict(rows=0), dict(vocab=0), dict(hidden=0), dict(ld_hidden=63), dict(ld_weight=56), dict(scale=-1.0), dict(states=at + 8), dict(ws=8)):
        refused(head(**bad), b"bb_head_logprob_fwd")
    room = handle.bb_grad_norm_workspace_bytes()
    one = lambda *fields: lib._tensor_table(1).pack(*fields)  # noqa: E731
    refused(handle.bb_grad_sumsq(None, 1, at, room, None), b"bb_grad_sumsq")
    refused(handle.bb_grad_sumsq(one(at, 4, 1, 0), 1, at, room - 1, None), b"bb_grad_sumsq")
    for fields, limit, ws in (((at, 4, 1, 0), 0.0, room), ((at, 0, 1, 0), 1.0, room), ((at + 2, 4, 1, 0), 1.0, room), ((at, 4, 2, 0), 1.0, room),
                              ((0, 4, 1, 0), 1.0, room), ((at, 4, 1, 0), 1.0, 8), ((at, 4, 1, 0), math.nan, room)):
        refused(handle.bb_grad_clip(one(*fields), 1, None, limit, at, at, ws, None), b"bb_grad_clip")
    for n, limit, ws in ((6, 1.0, room), (8, 0.0, room), (8, 1.0, 8)):
        refused(handle.bb_adam_step_clipped(at, at, at, at, None, n, 1e-3, 0.9, 0.999, 1e-8, 1, 1, 1, 0.0, 1.0, 1, None, limit, at, at, ws, None),
                b"bb_adam_step_clipped")


def test_descriptors_match_the_header():
    import re
    from bamboo_b200 import lib
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "bamboo_b200.h")).read()
    for name, struct in (("bb_preference_desc", lib.PreferenceDesc), ("bb_policy_desc", lib.PolicyDesc), ("bb_head_desc", lib.HeadDesc)):
        body = text[text.index(f"typedef struct {name}"):text.index(f"}} {name};")]
        fields = re.findall(r"(?:long long|int|double)\s+([a-z0-9_, ]+);", body)
        assert [f.strip() for group in fields for f in group.split(",")] == [n for n, _ in struct._fields_]
    assert lib._tensor_table(3).size == 3 * 24


def test_cpu_tensors_are_refused(monkeypatch):
    from bamboo_b200 import lib, post_training as pt
    x, t = torch.zeros(4, 16), torch.zeros(4, dtype=torch.int64)
    calls = (lambda: pt.token_logprobs(x, t), lambda: pt.head_logprobs(x.bfloat16(), x.bfloat16(), t),
             lambda: pt.preference_loss(x[:, 0].view(2, 2), None, t.view(2, 2)), lambda: pt.policy_loss(x[:, 0].view(2, 2), None, x[:, 0], t.view(2, 2)),
             lambda: pt.PreferenceLoss(16)(x, t), lambda: pt.PolicyLoss(16)(x, (t.view(2, 2), None, x[:, 0])), lambda: pt.clip_grad_norm_([x], 1.0),
             lambda: pt.adam_step_clipped(x, x, x, x, None, max_norm=1.0, lr=1.0, step=1))
    for call in calls:
        with pytest.raises(lib.BambooNativeError):
            call()
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    with pytest.raises(lib.BambooNativeError, match="current device"):         # another device's tensor is refused before a launch
        pt._on_current(type("OnThird", (), {"get_device": lambda self: 3})(), "x")
    import deepspeed.runtime.utils as ds_utils
    with pytest.raises(NotImplementedError):
        ds_utils.clip_grad_norm_([x], 1.0, norm_type=1)

"""``gradient_clipping`` with several engines over one store, one after the other and in turn: each clips by the norm of its own gradients."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from oracle import gpt_ref  # noqa: E402

CFG = gpt_ref.RefConfig(layers=4, hidden=32, heads=2, ffn=64, seq=8, vocab=48)
MB, GAS, LR, LIMIT = 2, 2, 1e-3, 0.5


def _engine(store, stages, seed):
    import cpu_layers
    from bamboo_b200 import api
    from bamboo_b200.module import PipelineModule
    model = PipelineModule(cpu_layers.ref_layer_specs(CFG, seed), num_stages=stages, loss_fn=cpu_layers.ref_loss(CFG),
                           partition_method="uniform", device="cpu")
    config = {"train_micro_batch_size_per_gpu": MB, "gradient_accumulation_steps": GAS, "gradient_clipping": LIMIT,
              "optimizer": {"type": "Adam", "params": {"lr": LR}}, "bamboo_b200": {"p2p_timeout_s": 20}}
    return api.initialize(model=model, config=config, redundancy_level=0, store=store)[0]


def _norms(engine, seed, steps):
    out = []
    for batches in gpt_ref.synthetic_batches(CFG, MB, GAS, steps, seed=seed):
        engine.train_batch(data_iter=iter(batches))
        out.append(engine.get_global_grad_norm())
    return out


def _train(rank, world, store):
    stages = world
    first = _norms(_engine(store, stages, 0), 1, 2)
    second = _engine(store, stages, 5)
    return first + _norms(second, 2, 2)


def test_engines_over_one_store_do_not_read_each_others_norms():
    from dist_utils import run_ranks
    os.environ["BAMBOO_QUIET"] = "1"
    want = _norms(_engine(None, 1, 0), 1, 2) + _norms(_engine(None, 1, 5), 2, 2)
    assert abs(want[0] - want[2]) > 1e-3 * want[0]
    res = run_ranks(_train, 2)
    for rank in range(2):
        assert res[rank][0] == "ok" and res[rank][1] == pytest.approx(want, rel=1e-4)

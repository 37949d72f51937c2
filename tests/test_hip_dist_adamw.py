"""Two ranks that share cuda:0 (gloo, collectives on host copies) train with FusedAdamW from the same averaged gradients: moments in
8 bits are rounded with random bits that do not depend on the rank, so both ranks hold the same parameters and states."""
import os
import shutil

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from conftest import GOLDEN, PKG
from test_hip_dist_trainer import _free_port

pytestmark = pytest.mark.gpu


def _worker(rank, port, root, strategy, optimizer, out):
    import sys
    sys.path.insert(0, PKG)
    import torch.distributed as dist
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    os.environ["GCN_UELB_MODEL_ROOT"] = os.path.join(root, "models")
    os.environ.pop("GCN_UELB_DATA_ROOT", None)
    try:
        dist.init_process_group("gloo", rank=rank, world_size=2)
        torch.cuda.set_device(0)
        from src.common.config.config import Settings
        from src.gcn.train.trainer import Trainer
        cfg = Settings(dict(data_root=root, dataset_name="nsf_small", packed_dataset=False, num_train_data=12, batch_size=4, num_nodes=14,
                            num_commodities=4, voc_edges_in=3, voc_edges_out=2 if strategy == "supervised" else 1, hidden_dim=64, num_layers=2,
                            mlp_layers=2, aggregation="mean", learning_rate=1e-3, max_epochs=1, training_strategy=strategy, beam_size=2, seed=5,
                            optimizer=optimizer, max_grad_norm=0.5))
        torch.manual_seed(100 + rank)
        trainer = Trainer(cfg, torch.float32, torch.long)
        before = torch.cat([p.detach().reshape(-1) for p in trainer.get_model().parameters()]).cpu().numpy()
        _, loss, _, _ = trainer.train_one_epoch()
        params = torch.cat([p.detach().reshape(-1) for p in trainer.get_model().parameters()]).cpu().numpy()
        states = [(k, st[k].cpu().numpy()) for st in trainer.optimizer.state.values() for k in sorted(st) if k != "step"]
        out.put((rank, "ok", float(loss), before, params, states))
    except Exception as ex:  # pragma: no cover
        import traceback
        out.put((rank, "error: " + repr(ex) + traceback.format_exc()[-1500:], 0.0, None, None, None))
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


@pytest.mark.parametrize("strategy,optimizer", [("supervised", "adamw8bit"), ("supervised", "adamw"), ("reinforcement", "adamw8bit")])
def test_two_ranks_hold_the_same_parameters_and_states(strategy, optimizer, tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    shutil.copytree(os.path.join(GOLDEN, "datasets", "nsf_small"), tmp_path / "nsf_small")
    ctx = mp.get_context("spawn")
    out, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, port, str(tmp_path), strategy, optimizer, out)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted([out.get(timeout=100) for _ in procs], key=lambda r: r[0])
    for p in procs:
        p.join(timeout=30)
    assert [r[1] for r in res] == ["ok", "ok"], res
    (_, _, loss, before, params, states), (_, _, _, _, other_params, other_states) = res
    assert np.isfinite(loss) and np.isfinite(params).all() and not np.array_equal(before, params)
    assert np.array_equal(params, other_params)
    assert [k for k, _ in states] == [k for k, _ in other_states]
    assert any(x.dtype == np.uint8 for _, x in states) == (optimizer == "adamw8bit")      # 64 x 64 weights: 4096 elements
    assert all(np.array_equal(a, b) for (_, a), (_, b) in zip(states, other_states))

"""Link score rules and the trainer's choice of optimizer: what needs no GPU."""
import pytest
import torch

from src.common.config.config import Settings
from src.gcn.algorithms.score_rules import LinkScoreRules, hops_from
from src.gcn.hip.lib import GcnHipError


def test_hops_from_paths():
    paths = torch.tensor([[[0, 2, 1, -1], [3, 1, -1, -1], [2, -1, -1, -1]], [[1, 0, 3, 2], [9, 1, 2, -1], [0, 3, 1, 2]]], dtype=torch.int32)
    length = torch.tensor([[3, 2, 1], [4, 3, 2]], dtype=torch.int32)
    hops = hops_from(paths, length, 4)
    want = torch.full((2, 4, 3), -1)
    for b in range(2):
        for k in range(3):
            row = paths[b, k, :length[b, k]].tolist()
            for here, there in zip(row, row[1:]):
                if 0 <= here < 4 and 0 <= there < 4:
                    want[b, here, k] = there
    assert hops.dtype == torch.int32 and hops.is_contiguous() and torch.equal(hops.long(), want)
    assert hops_from(paths[:, :, :1], length.clamp(max=1), 4).eq(-1).all()


def test_refusals():
    with pytest.raises(GcnHipError):
        LinkScoreRules(torch.ones(1, 3, 3))


def test_trainer_optimizer_choice():
    from src.gcn.hip.fused_adam import FusedAdam
    from src.gcn.hip.fused_adamw import FusedAdamW
    from src.gcn.train.trainer import make_optimizer
    p = lambda: [torch.nn.Parameter(torch.ones(3))]
    assert type(make_optimizer(Settings(dict(learning_rate=1e-3)), p())) is FusedAdam
    opt = make_optimizer(Settings(dict(learning_rate=1e-3, optimizer="adamw")), p())
    assert type(opt) is FusedAdamW and opt.state_bits == 32 and opt.param_groups[0]["weight_decay"] == 0.01 and opt.max_grad_norm is None
    opt = make_optimizer(Settings(dict(learning_rate=1e-3, optimizer="adamw8bit", weight_decay=0.1, max_grad_norm=2.0)), p())
    assert opt.state_bits == 8 and opt.param_groups[0]["weight_decay"] == 0.1 and opt.max_grad_norm == 2.0
    with pytest.raises(ValueError, match="adamw8bit"):
        make_optimizer(Settings(dict(learning_rate=1e-3, optimizer="sgd")), p())

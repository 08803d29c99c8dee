"""Which clipping norm a training step uses: the caller's, else the optimizer's own, else the reference trainer's 1.0."""
from types import SimpleNamespace

import pytest
import torch

from recommend_amd.dist_train import ShardedTrainStep
from recommend_amd.optim import FusedAdamW, FusedClipAdam

MODEL = SimpleNamespace(group=None, world=1, rank=0, parameters=lambda: [torch.nn.Parameter(torch.zeros(2))])


@pytest.mark.parametrize("optimizer", [FusedAdamW, FusedClipAdam])
@pytest.mark.parametrize("own,given,want", [(0.3, {}, 0.3), (None, {}, 1.0), (0.3, {"max_grad_norm": 2.0}, 2.0),
                                            (0.3, {"max_grad_norm": None}, None), (0.0, {}, 0.0)])
def test_an_optimizer_that_clips_keeps_its_own_norm(optimizer, own, given, want):
    opt = optimizer([torch.nn.Parameter(torch.zeros(2))], max_grad_norm=own)
    step = ShardedTrainStep(MODEL, opt, None, **given)
    assert opt.max_grad_norm == step.max_grad_norm == want


@pytest.mark.parametrize("given,want", [({}, 1.0), ({"max_grad_norm": 2.0}, 2.0), ({"max_grad_norm": None}, None)])
def test_an_optimizer_that_does_not_clip_is_left_alone(given, want):
    opt = torch.optim.SGD([torch.nn.Parameter(torch.zeros(2))], lr=0.1)
    assert ShardedTrainStep(MODEL, opt, None, **given).max_grad_norm == want and not hasattr(opt, "max_grad_norm")

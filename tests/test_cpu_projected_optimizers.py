"""What ``ProjectedFusedStep.update`` steps: the optimizer or optimizers that the object holds now."""
from types import SimpleNamespace

import pytest
import torch


class _Counts(torch.optim.SGD):
    steps = 0

    def step(self, closure=None):
        self.steps += 1


@pytest.fixture
def parts():
    from haste_b200.norm import LayerNorm
    lin, norm = torch.nn.Linear(8, 16, dtype=torch.bfloat16), LayerNorm(16)
    return lin, norm, SimpleNamespace(D=16), lambda params: _Counts(list(params), lr=1.0)


def test_one_and_several(parts):
    from haste_b200.projected import ProjectedFusedStep
    lin, norm, shard, make = parts
    one = make([*lin.parameters(), *norm.parameters()])
    ProjectedFusedStep(lin, norm, shard, one).update()
    assert one.steps == 1
    several = [make([lin.weight]), make([lin.bias, *norm.parameters()])]
    for held in (several, tuple(several)):
        ProjectedFusedStep(lin, norm, shard, held).update()
    assert [o.steps for o in several] == [2, 2]
    with pytest.raises(ValueError):
        ProjectedFusedStep(lin, norm, shard, several[:1])


def test_replaced(parts):
    from haste_b200.projected import ProjectedFusedStep
    lin, norm, shard, make = parts
    first, second = (make([*lin.parameters(), *norm.parameters()]) for _ in range(2))
    step = ProjectedFusedStep(lin, norm, shard, first)
    step.optimizer = second
    step.update()
    step.optimizer = [first, second]
    step.update()
    assert (first.steps, second.steps) == (1, 2)

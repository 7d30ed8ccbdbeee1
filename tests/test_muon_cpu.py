"""Refusals of the Muon operators that need no GPU."""

import pytest
import torch

from synthefy_nori_b200 import ops


def test_newton_schulz_refuses_cpu_tensors():
    for g in (torch.zeros(4, 4), torch.zeros(4), [[1.0]]):
        with pytest.raises(ValueError):
            ops.newton_schulz(g)


@pytest.mark.parametrize("shapes,offsets,moff", [
    ([(4, 4)], [0, 16], None),                      # one offset too many
    ([(4, 4)], [0], [0, 16]),
    ([(4, 4)], [-1], None),
    ([(4, 4)], [0], [-4]),
    ([(0, 4)], [0], None),
    ([(4, 1 << 20)], [0], None),
    ([(4, 4), (4, 4)], [0, 0], None),               # the same matrix twice
    ([(4, 4), (2, 2)], [0, 15], None),              # overlap by one value
    ([(4, 4), (2, 2)], [0, 16], [0, 15]),
])
def test_plan_refuses(shapes, offsets, moff):
    with pytest.raises(ValueError):
        ops.MuonPlan(shapes, offsets, "cuda", moff)


def test_plan_refuses_cpu_device():
    with pytest.raises(ValueError):
        ops.MuonPlan([(4, 4)], [0], "cpu")


def test_muon_step_refuses_cpu_buffers():
    class Plan:
        extent = momentum_extent = 16

    z = torch.zeros(16)
    with pytest.raises(ValueError):
        ops.muon_step(Plan(), z, z, z, lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_step(Plan(), z, z, z, lr=0.1, adjust_lr="other")

"""An optimizer step raises the version counter of every parameter it may have changed: caches of
derived weights and autograd's check of saved tensors read it."""

import pytest
import torch

from synthefy_nori_b200.training.muon import HybridMuonAdamW
from synthefy_nori_b200.training.optim import FlatParams, FusedAdamWEMA


def _net():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(6, 5), torch.nn.LayerNorm(5), torch.nn.Linear(5, 3))


@pytest.mark.parametrize("kind", ["adamw", "muon"])
def test_step_raises_every_parameter(kind):
    net = _net()
    opt = HybridMuonAdamW(net, "cpu") if kind == "muon" else FusedAdamWEMA(FlatParams(net.parameters(), "cpu"))
    opt.flat.grad.normal_()
    before = [p._version for p in net.parameters()]
    opt.step()
    assert all(p._version > v for p, v in zip(net.parameters(), before))


@pytest.mark.parametrize("kind", ["adamw", "muon"])
def test_backward_after_a_step_is_refused(kind):
    """Weights that changed between the forward and the backward pass."""
    net = _net()
    opt = HybridMuonAdamW(net, "cpu") if kind == "muon" else FusedAdamWEMA(FlatParams(net.parameters(), "cpu"))
    x = torch.randn(4, 6, requires_grad=True)
    y = net(x).sum()
    opt.flat.grad.normal_()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()

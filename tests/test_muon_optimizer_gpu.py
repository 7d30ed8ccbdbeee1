"""HybridMuonAdamW on the GPU beside its kernels: rejected steps without a plan, matrices without
values, and the kernels against the exact iteration with nothing else in their place."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("skip", [None, 0.0, 1.0])
@pytest.mark.parametrize("ns_steps", [0, 5])
def test_gradient_norm_that_is_not_finite(bad, skip, ns_steps):
    """With the kernels and without (no iteration at all is not theirs)."""
    from synthefy_nori_b200.training.muon import HybridMuonAdamW

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(6, 5), torch.nn.Linear(5, 300)).cuda()
    opt = HybridMuonAdamW(net, "cuda", lr=0.1, max_grad_norm=1.0, ns_steps=ns_steps)
    assert (opt.plan is None) == (ns_steps == 0)

    def state():
        sd = opt.state_dict()
        return [opt.flat.data, sd["m"], sd["v"], sd["ema"], *sd["muon_momentum"]]

    sk = None if skip is None else torch.tensor(skip, device="cuda")
    opt.flat.grad.normal_()
    opt.step()
    before = copy.deepcopy(state())
    opt.flat.grad[3] = bad
    opt.step(skip=sk)
    assert all(torch.equal(a, b) for a, b in zip(before, state()))
    opt.flat.grad.normal_()
    opt.step()
    assert not any(torch.equal(a, b) for a, b in zip(before, state()))
    assert all(t.isfinite().all() for t in state())


def test_matrices_without_values():
    from synthefy_nori_b200.training.muon import HybridMuonAdamW

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.b = torch.nn.Parameter(torch.randn(7, 6))
            self.c = torch.nn.Parameter(torch.randn(0, 6))

    torch.manual_seed(1)
    net = Net().cuda()
    opt = HybridMuonAdamW(net, "cuda", lr=0.1)
    assert opt.plan is not None and opt.plan.count == 1
    before = net.b.detach().clone()
    opt.flat.grad.normal_()
    opt.step()
    assert not torch.equal(before, net.b) and net.b.isfinite().all()
    assert [tuple(t.shape) for t in opt.state_dict()["muon_momentum"]] == [(1, 7, 6), (1, 0, 6)]


def test_step_runs_the_kernels_alone(monkeypatch):
    """No other orthogonalisation is called, and the weights are those of the 64-bit iteration."""
    from test_muon_steps_gpu import iterate64, tolerance

    from synthefy_nori_b200.training import muon as tm

    torch.manual_seed(2)
    net = torch.nn.Sequential(torch.nn.Linear(48, 96), torch.nn.GELU(), torch.nn.Linear(96, 260)).cuda()
    opt = tm.HybridMuonAdamW(net, "cuda", lr=0.01, weight_decay=0.1, max_grad_norm=0.05)
    assert opt.plan is not None and opt.plan.count == 2

    def unused(*a, **k):
        raise AssertionError("newton_schulz called beside the step")

    monkeypatch.setattr(tm, "newton_schulz", unused)
    opt.zero_grad()
    net(torch.randn(64, 48, device="cuda")).square().mean().backward()
    clip = min(1.0, 0.05 / (float(opt.flat.grad.double().norm()) + 1e-6))
    before = {k: (p.detach().double().clone(), p.grad.double().clone()) for k, p in net.named_parameters()}
    opt.step()
    for k, p in net.named_parameters():
        if p.ndim < 2:
            continue
        w, g = before[k]
        u = 1.95 * clip * g  # the first step's gradient and momentum
        upd = 0.01 * 0.2 * max(w.shape) ** 0.5 * iterate64(u[None], 5)[0]
        tol = tolerance(u, 5) * float(upd.norm()) + 4 * 2.0 ** -24 * float(w.norm() + upd.norm())
        assert float((p.detach().double() - (w * (1 - 0.01 * 0.1) - upd)).norm()) < tol, k

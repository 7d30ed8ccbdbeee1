"""Native optimizer steps and what is derived from the weights they change."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _optimizer(kind, model):
    from synthefy_nori_b200.training.muon import HybridMuonAdamW
    from synthefy_nori_b200.training.optim import FlatParams, FusedAdamWEMA

    if kind == "adamw":
        return FusedAdamWEMA(FlatParams(model.parameters(), "cuda"), lr=0.02)
    opt = HybridMuonAdamW(model, "cuda", lr=0.02, include_nd=True)
    assert opt.plan is not None
    return opt


@pytest.mark.parametrize("kind", ["muon", "adamw"])
def test_two_phase_inference_follows_the_optimizer(kind):
    """Evaluate, step, evaluate: the second answer is the one of a fresh model with these weights."""
    from synthefy_nori_b200.models.config import preset_config
    from synthefy_nori_b200.utils.loading import build_model

    cfg = preset_config("nori-tiny")
    cfg["two_phase_config"] = {"target_tokens": 2, "row_layers": 1, "row_heads": 2, "row_hidden_dim": 96}
    torch.manual_seed(0)
    model = build_model(cfg).cuda().eval()
    opt = _optimizer(kind, model)
    x, y = torch.randn(1, 90, 6, device="cuda"), torch.randn(1, 60, device="cuda")

    def answer(m):
        with torch.no_grad():
            assert m.use_native_two_phase(x.device)
            return m(x, y, 60, task_type="reg")

    first = answer(model)
    opt.flat.grad.normal_()
    opt.step()
    second = answer(model)
    fresh = build_model(cfg).cuda().eval()
    fresh.load_state_dict(model.state_dict())
    assert torch.equal(second, answer(fresh))
    assert not torch.equal(first, second)


@pytest.mark.parametrize("kind", ["muon", "adamw"])
def test_step_raises_every_parameter(kind):
    net = torch.nn.Sequential(torch.nn.Linear(6, 200), torch.nn.LayerNorm(200), torch.nn.Linear(200, 300)).cuda()
    opt = _optimizer(kind, net)
    y = net(torch.randn(4, 6, device="cuda", requires_grad=True)).sum()
    opt.flat.grad.normal_()
    before = [p._version for p in net.parameters()]
    opt.step()
    assert all(p._version > v for p, v in zip(net.parameters(), before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_operators_raise_what_they_write():
    from synthefy_nori_b200 import ops

    g = torch.randn(20, 12, device="cuda")
    out = torch.empty_like(g)
    v, w = g._version, out._version
    ops.newton_schulz(g, out=out)
    assert out._version > w and g._version == v
    data, grad, mom, ema = (torch.randn(240, device="cuda") for _ in range(4))
    before = [t._version for t in (data, grad, mom, ema)]
    ops.muon_step(ops.MuonPlan([(20, 12)], [0], "cuda"), data, grad, mom, lr=0.1, ema=ema)
    after = [t._version for t in (data, grad, mom, ema)]
    assert [a > b for a, b in zip(after, before)] == [True, False, True, True]

"""The native encoder's and head's copies of the weights follow every in-place change of them."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _build():
    from synthefy_nori_b200.models.config import preset_config
    from synthefy_nori_b200.utils.loading import build_model

    return build_model(preset_config("nori-tiny")).cuda().eval()


@pytest.mark.parametrize("change", ["muon", "adamw", "in place", "torch optimizer"])
@pytest.mark.parametrize("inference", [False, True])
def test_native_inference_follows_the_weights(change, inference):
    from synthefy_nori_b200.training.muon import HybridMuonAdamW
    from synthefy_nori_b200.training.optim import FlatParams, FusedAdamWEMA

    torch.manual_seed(0)
    model = _build()
    x, y = torch.randn(1, 90, 6, device="cuda"), torch.randn(1, 60, device="cuda")
    mode = torch.inference_mode if inference else torch.no_grad
    if change == "muon":
        opt = HybridMuonAdamW(model, "cuda", lr=0.05, include_nd=True)
        assert opt.plan is not None
    elif change == "adamw":
        opt = FusedAdamWEMA(FlatParams(model.parameters(), "cuda"), lr=0.05)
    elif change == "torch optimizer":
        opt = torch.optim.SGD(model.parameters(), lr=0.05)

    def answer(m):
        with mode():
            return m(x, y, 60, task_type="reg")

    first = answer(model)
    assert torch.equal(first, answer(model))
    if change == "in place":
        with torch.no_grad():
            for p in model.parameters():
                p.add_(0.05 * torch.randn_like(p))
    else:
        for p in model.parameters():
            if p.requires_grad:
                p.grad = torch.randn_like(p) if change == "torch optimizer" else p.grad.normal_()
        opt.step()
    second = answer(model)
    fresh = _build()
    fresh.load_state_dict(model.state_dict())
    assert torch.equal(second, answer(fresh))
    assert not torch.equal(first, second)

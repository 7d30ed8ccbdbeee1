"""The training operators as a run uses them: LayerNorm encoder layers on the module path,
their gradients, and a Muon step on what they give."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _layers(pre_norm, arch):
    from synthefy_nori_b200.models.layers import EncoderBaseLayer, LayerNorm

    torch.manual_seed(0)
    net = torch.nn.Sequential()
    for i in range(2):
        net.add_module(f"l{i}", EncoderBaseLayer(nhead=2, embed_dim=32, hid_dim=48, pre_norm=pre_norm, layer_arch=arch,
                                                 seq_attn_isolated=True))
    net.add_module("norm", LayerNorm(32))
    return net


def _forward(net, x, eval_pos):
    for m in list(net)[:-1]:
        x = m(x, eval_pos=eval_pos)[0]
    return net[-1](x)


@pytest.mark.parametrize("pre_norm", [True, False])
@pytest.mark.parametrize("arch", ["smf", "fmfmsm"])
def test_layer_norm_layers_train_with_muon(pre_norm, arch):
    from synthefy_nori_b200.training.muon import HybridMuonAdamW

    net = _layers(pre_norm, arch)
    ref = copy.deepcopy(net).double()
    net = net.cuda()
    opt = HybridMuonAdamW(net, "cuda", lr=1e-3, include_nd=True, max_grad_norm=1.0)
    assert opt.plan is not None
    x = torch.randn(2, 12, 5, 32)
    c = torch.randn(2, 12, 5, 32)
    opt.zero_grad()
    y = _forward(net, x.cuda(), 8)
    (y * c.cuda()).sum().backward()
    want = _forward(ref, x.double(), 8)
    (want * c.double()).sum().backward()
    # fp32 against 64 bits through two layers: products of 32 to 96 terms, each sum within 2^-17
    assert float((y.cpu().double() - want).detach().norm() / want.detach().norm()) < 2.0 ** -14
    for (name, p), r in zip(net.named_parameters(), ref.parameters()):
        if r.grad is not None:
            assert float((p.grad.cpu().double() - r.grad).norm()) < 2.0 ** -12 * float(r.grad.norm()) + 1e-5, name
    before = [p.detach().clone() for p in net.parameters()]
    for _ in range(3):
        opt.step(skip=torch.zeros((), device="cuda"))
    moved = [float((p.detach() - b).norm()) for p, b, r in zip(net.parameters(), before, ref.parameters()) if r.grad is not None]
    assert all(0 < m < float("inf") for m in moved)


def test_layer_norm_module_in_inference_mode_and_checkpoint():
    from torch.utils.checkpoint import checkpoint

    from synthefy_nori_b200.models.layers import LayerNorm

    torch.manual_seed(1)
    m = LayerNorm(40).cuda()
    x = torch.randn(7, 40, device="cuda")
    want = m(x).detach()
    with torch.inference_mode():
        assert torch.equal(m(x), want)
    with torch.no_grad():
        assert torch.equal(m(x), want)
    a = x.clone().requires_grad_(True)
    b = x.clone().requires_grad_(True)
    m(a).square().sum().backward()
    ga, m.weight.grad = m.weight.grad, None
    checkpoint(m, b, use_reentrant=False).square().sum().backward()
    assert torch.equal(a.grad, b.grad) and torch.equal(ga, m.weight.grad)

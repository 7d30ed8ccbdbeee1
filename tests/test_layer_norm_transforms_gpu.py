"""Function transforms, forward-mode derivatives and tracing of the model's LayerNorm modules on CUDA
give what torch's module gives."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _pair(width=24):
    from synthefy_nori_b200.models.layers import LayerNorm

    torch.manual_seed(0)
    m, t = LayerNorm(width).cuda(), torch.nn.LayerNorm(width).cuda()
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    t.load_state_dict(m.state_dict())
    return m, t, torch.randn(6, 5, width, device="cuda")


def test_func_grad_vmap_and_jvp():
    m, t, x = _pair()
    f = torch.func
    for run in (lambda n: f.grad(lambda v: n(v).square().sum())(x), lambda n: f.vmap(n)(x),
                lambda n: f.jvp(n, (x,), (x.cos(),))[1], lambda n: f.vjp(n, x)[1](x.sin())[0],
                lambda n: f.vmap(f.grad(lambda v: n(v).sin().sum()))(x)):
        assert torch.equal(run(m), run(t))
    params = dict(m.named_parameters())
    loss = lambda n: lambda p: f.functional_call(n, p, (x,)).square().sum()  # noqa: E731
    a, b = f.grad(loss(m))(params), f.grad(loss(t))(params)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_forward_mode_dual_numbers():
    import torch.autograd.forward_ad as fw

    m, t, x = _pair()
    with fw.dual_level():
        d = fw.make_dual(x, x.cos())
        a, b = fw.unpack_dual(m(d)), fw.unpack_dual(t(d))
        assert torch.equal(a.primal, b.primal) and torch.equal(a.tangent, b.tangent)


def test_traced_module_follows_its_input():
    m, t, x = _pair()
    with torch.no_grad():
        traced = torch.jit.trace(m, x)
        assert torch.equal(traced(2 * x + 1), t(2 * x + 1))


def test_exported_module_follows_its_input():
    m, t, x = _pair()
    program = torch.export.export(m, (x,))
    with torch.no_grad():
        assert torch.equal(program.module()(2 * x + 1), t(2 * x + 1))


def test_fake_forward_and_backward():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from synthefy_nori_b200.models.layers import LayerNorm

    with FakeTensorMode():
        m, x = LayerNorm(24, device="cuda"), torch.empty(5, 24, device="cuda", requires_grad=True)
        m(x).sum().backward()
        assert x.grad.shape == x.shape and m.weight.grad.shape == (24,)


def test_real_tensors_under_a_fake_mode_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from synthefy_nori_b200 import ops

    x = torch.randn(6, 200, 300, device="cuda")
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(RuntimeError, match="plain tensor"):
            ops.layer_norm_fwd(x[0])
        with pytest.raises(RuntimeError, match="plain tensor"):
            ops.newton_schulz(x)
        with pytest.raises(RuntimeError, match="plain tensor"):
            ops.newton_schulz(x[:, :20, :10].contiguous())
    assert torch.equal(ops.newton_schulz(x), ops.newton_schulz(x))  # the status word is a real one

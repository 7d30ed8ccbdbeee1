"""Query passes over a block-scaled cache with a learnable temperature."""

import pytest
import torch

from test_block_cache_model_gpu import TYPES, _close, _model, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.0, -0.5, 2.0])
@pytest.mark.parametrize("nq", [1, 100])
@pytest.mark.parametrize("kw", [{}, dict(placement="stream", stream_block_rows=128)], ids=["resident", "stream"])
def test_any_temperature(dtype, temperature, nq, kw):
    """Its magnitude counts; 0 makes all keys equal."""
    m = _model(use_learnable_attn_temperature=True)
    for name, p in m.named_parameters():
        if "attn_temperature" in name:
            p.data.fill_(temperature)
    x, y = _table()
    with torch.no_grad():
        want = m.apply_context_cache(x[:, 300 : 300 + nq], m.build_context_cache(x[:, :300], y[:, :300]))
        got = m.apply_context_cache(x[:, 300 : 300 + nq], m.build_context_cache(x[:, :300], y[:, :300], cache_dtype=dtype, **kw))
    assert torch.isfinite(got).all()
    _close(got, want, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq", [1, 150])
def test_temperature_zero_is_the_mean(dtype, nq):
    from synthefy_nori_b200.ops import fused_layer as fl

    g = fl.Geometry(B=2, ep=333, nq=nq, T=3, E=112, H=2)
    kv = torch.randn(g.R_ctx, 2 * g.A, device="cuda").to(torch.bfloat16)
    q = (100 * torch.randn(g.R_q, g.A, device="cuda")).to(torch.bfloat16)
    cache = fl.BlockKV.empty(g, dtype, g.H, "cuda").write(kv)
    o = torch.empty_like(q)
    lse = cache.attend(q, o, g, 0.0, return_lse=True)
    v = cache.dequantize()[:, g.A :].double().view(2, 333, 3, g.A)
    want = v.mean(1, keepdim=True).expand(-1, nq, -1, -1)
    # half a step; weights to fp16, values to bf16 by dequantize
    size = v.abs().mean(1, keepdim=True)
    assert ((o.double().view(2, nq, 3, g.A) - want).abs() <= want.abs() * 2.0 ** -8 + size * (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -8)).all()
    assert (lse.double() - torch.log(torch.tensor(333.0, dtype=torch.float64))).abs().max() <= 2.0 ** -13

"""LayerNorm operator without a GPU: refusals, and the model's modules on their CPU path."""

import pytest
import torch

from synthefy_nori_b200 import ops


def test_refuses_cpu_tensors():
    x = torch.randn(4, 8)
    with pytest.raises(ValueError):
        ops.layer_norm(x)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, x, x[:, 0], x[:, 0])


def test_modules_on_the_cpu_are_torchs():
    from synthefy_nori_b200.models.layers import LayerNorm, LayerNormMixedPrecision

    torch.manual_seed(0)
    x = torch.randn(3, 5, 24)
    for cls in (LayerNorm, LayerNormMixedPrecision):
        m, t = cls(24), torch.nn.LayerNorm(24)
        assert isinstance(m, torch.nn.LayerNorm) and list(m.state_dict()) == list(t.state_dict())
        assert torch.equal(m(x), t(x))


def test_model_norms_are_the_module():
    from synthefy_nori_b200.models.config import base_config, finalize_arch_config, set_regression_head
    from synthefy_nori_b200.models.layers import LayerNorm
    from synthefy_nori_b200.utils.loading import build_model

    cfg = finalize_arch_config(set_regression_head(base_config()))
    m = build_model(cfg)
    norms = [x for x in m.modules() if isinstance(x, torch.nn.LayerNorm)]
    assert norms and all(isinstance(x, LayerNorm) for x in norms)

"""Builds of a block-scaled context cache in chunks of rows, as long contexts are built where memory is short."""

import pytest
import torch

from test_block_cache_model_gpu import TYPES, _model, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 100, 200, 257, 640, 699])
def test_codes_do_not_depend_on_the_chunk(dtype, rows, monkeypatch):
    """Whatever number of rows fits the free memory: the first layer's codes and scales (whose inputs no chunk
    changes) are those of a build in one pass."""
    from synthefy_nori_b200.ops import fused_layer

    m = _model()
    x, y = _table(B=1, rows=700)
    with torch.no_grad():
        full = m.build_context_cache(x, y, cache_dtype=dtype).caches
        monkeypatch.setattr(fused_layer, "_build_rows_chunk", lambda *a: rows)
        part = m.build_context_cache(x, y, cache_dtype=dtype).caches
    a, b = (c[0]["seq_kv"] for c in (full, part))
    for s, t in zip(a.cache[2:4], b.cache[2:4]):
        assert torch.equal(s[:, :, :11], t[:, :, :11])  # (blocks of rows that are there)
    for s, t in zip(a.cache[:2], b.cache[:2]):
        assert torch.equal(s[:, :, :700].view(torch.int8), t[:, :, :700].view(torch.int8))
    # every later layer: the same values but for what its inputs' rounding to bf16 makes of them
    for c, d in zip(full[1:], part[1:]):
        s, t = (z["seq_kv"].dequantize().float() for z in (c, d))
        assert torch.nn.functional.cosine_similarity(s.flatten(), t.flatten(), dim=0) > 0.999

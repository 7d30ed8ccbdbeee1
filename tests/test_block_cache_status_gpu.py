"""What block-scaled attention does once a wait on the device has run out (the status word says so)."""

import pytest
import torch

from test_block_attention_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,rows", [(200, 100), (1100, 128)])
def test_after_a_timeout_many_rows_are_left_alone(n, rows):
    """Whole CTAs leave, their tensor memory freed: nothing is written, and calls work again once the word is cleared."""
    from synthefy_nori_b200 import ops

    cache, g = make(3, 4, rows, 56)
    q = torch.randn(3, n, 4, 56, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    word = ops.status_word(q.device)
    try:
        word.fill_(2)
        for _ in range(3):
            ops.block_cache_attention(q, cache, rows, out=out)
        with pytest.raises(RuntimeError, match="timeout"):
            ops.check_status(q.device)
    finally:
        word.zero_()
    assert (out == 7.0).all()
    for _ in range(3):
        check(q, cache, [rows] * 3, ops.block_cache_attention(q, cache, rows, out=out))
    ops.check_status(q.device)


@pytest.mark.parametrize("n,rows", [(200, 700), (1100, 3000), (1, 100003)])
def test_after_a_timeout_no_parts_are_joined(n, rows):
    """Where the keys are split, the join does not read parts that were never written."""
    from synthefy_nori_b200 import ops

    cache, g = make(1, 2, rows, 56)
    q = torch.randn(1, n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    word = ops.status_word(q.device)
    try:
        word.fill_(2)
        for _ in range(3):
            ops.block_cache_attention(q, cache, rows, out=out)
    finally:
        word.zero_()
    assert (out == 7.0).all()
    check(q, cache, [rows], ops.block_cache_attention(q, cache, rows, out=out))


@pytest.mark.parametrize("call", ["predict", "embeddings", "build"])
def test_a_timeout_reaches_who_predicts(call, monkeypatch):
    """A wait that ran out in a query pass or a build is an error, and nothing of that build is kept."""
    import numpy as np

    from synthefy_nori_b200 import NoriRegressor, ops

    rng = np.random.default_rng(0)
    X = rng.normal(size=(200, 4)).astype(np.float32)
    r = NoriRegressor(model="nori-tiny", weights="random", device="cuda", n_estimators=1, cache_dtype="block_int8")
    r.fit(X[:150], X[:150, 0])
    want = r.predict(X[150:])
    pred, word = r.predictor_, ops.status_word(torch.device("cuda", torch.cuda.current_device()))
    name = "build_context_cache" if call == "build" else "apply_context_cache"
    stock = getattr(pred.model, name)

    def fails(*a, **kw):
        res = stock(*a, **kw)
        word.fill_(3)  # as a kernel of the call would have set it
        return res

    try:
        with monkeypatch.context() as m:
            m.setattr(pred.model, name, fails)
            with pytest.raises(RuntimeError, match="timeout"):
                if call == "build":
                    pred.fit_context(X[:100], X[:100, 0])
                elif call == "predict":
                    r.predict(X[150:])
                else:
                    r.get_embeddings(X[150:])
    finally:
        word.zero_()
    if call == "build":
        hits = pred.store.hits
        pred.fit_context(X[:100], X[:100, 0])
        assert pred.store.hits == hits
    assert np.array_equal(r.predict(X[150:]), want)


FIRST_CALL = """
import torch
from synthefy_nori_b200 import ops

cache = ops.block_cache(2, 2, 640, 32)
x = torch.randn(2, 640, 2, 32, device="cuda")
ops.block_cache_write(cache, x, x)
q = torch.randn(2, 200, 2, 32, device="cuda").to(torch.bfloat16)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):  # the first call that takes the word
    o = ops.block_cache_attention(q, cache, 640)
assert int(ops.status_word(q.device).item()) == 0
graph.replay()
want = ops.block_cache_attention(q, cache, 640)
assert torch.equal(o, want)
word = ops.status_word(q.device)
word.fill_(7)
o.zero_()
graph.replay()
assert int(word.item()) == 7 and not o.any()
word.zero_()
graph.replay()
assert torch.equal(o, want)
print("fine")
"""


def test_the_first_call_may_be_captured():
    """The status word is not part of the graph that happens to make the first call: replays do not clear it."""
    import subprocess
    import sys

    run = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "fine" in run.stdout, run.stderr[-2000:]

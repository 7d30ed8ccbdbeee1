"""LayerNorm with weights of other types than fp32, and its autograd node, against the formulas in 64
bits (tolerances as for fp32 weights: a 16-bit weight is exact in fp32)."""

import pytest
import torch
from test_layer_norm_gpu import check

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("tx,tw,tb", [(BF, BF, BF), (HF, HF, HF), (BF, BF, F32), (BF, F32, BF), (F32, BF, BF), (HF, BF, HF),
                                      (BF, torch.float64, None), (F32, None, HF)])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 5), (37, 64), (300, 56), (70, 448), (33, 999), (9, 2500), (3, 9001)])
def test_weights_of_each_type(tx, tw, tb, rows, cols):
    from synthefy_nori_b200 import ops

    torch.manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda").to(tx)
    w = None if tw is None else (1 + 0.3 * torch.randn(cols, device="cuda")).to(tw)
    b = None if tb is None else torch.randn(cols, device="cuda").to(tb)
    if tw == torch.float64:
        w = w.float().double()  # (cast to fp32 on the way)
    check(x, w, b, torch.randn(rows, cols, device="cuda").to(tx), None, ops)
    if tx != F32:
        check(x, w, b, torch.randn(rows, cols, device="cuda"), F32, ops)


@pytest.mark.parametrize("tx", [BF, HF])
@pytest.mark.parametrize("cols", [64, 57])
def test_weights_off_their_alignment_and_strided(tx, cols):
    from synthefy_nori_b200 import ops

    torch.manual_seed(1)
    x, dy = torch.randn(50, cols, device="cuda").to(tx), torch.randn(50, cols, device="cuda").to(tx)
    wide = torch.randn(2 * cols + 1, device="cuda").to(tx)
    check(x, wide[1 : cols + 1], wide[:cols], dy, None, ops)
    check(x, wide[: 2 * cols : 2], wide[1 : 2 * cols : 2], dy, None, ops)


@pytest.mark.parametrize("tx,tw", [(BF, BF), (HF, HF), (BF, F32), (F32, BF), (F32, F32)])
@pytest.mark.parametrize("shape", [(2, 3, 40), (5000, 40), (7, 700), (2, 9000)])
@pytest.mark.parametrize("out", [None, F32])
def test_node_gives_the_operators_gradients(tx, tw, shape, out):
    from synthefy_nori_b200 import ops

    torch.manual_seed(2)
    C = shape[-1]
    x = torch.randn(shape, device="cuda").to(tx).requires_grad_(True)
    w = torch.randn(C, device="cuda").to(tw).requires_grad_(True)
    b = torch.randn(C, device="cuda").to(tw).requires_grad_(True)
    y = ops.layer_norm(x, w, b, out_dtype=out)
    z, mean, rstd = ops.layer_norm_fwd(x.detach(), w.detach(), b.detach(), out_dtype=out)
    assert torch.equal(y, z) and y.dtype == (out or tx)
    dy = torch.randn(shape, device="cuda").to(y.dtype)
    got = torch.autograd.grad(y, (x, w, b), dy)
    want = ops.layer_norm_bwd(dy, x.detach(), mean, rstd, w.detach())
    for g, r, t in zip(got, want, (x, w, b)):
        assert g.dtype == t.dtype and g.shape == t.shape and torch.equal(g, r.to(t.dtype))
    with torch.no_grad():
        q = ops.layer_norm(x, w, b, out_dtype=out)
    assert torch.equal(q, z) and not q.requires_grad


def test_node_with_some_inputs_wanted():
    from synthefy_nori_b200 import ops

    torch.manual_seed(3)
    x, w, b = (torch.randn(s, device="cuda") for s in ((9, 24), (24,), (24,)))
    dy = torch.randn(9, 24, device="cuda")
    _, mean, rstd = ops.layer_norm_fwd(x, w)
    want = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    plain = ops.layer_norm_bwd(dy, x, mean, rstd, None)
    for wanted in range(1, 8):
        t = [v.clone().requires_grad_(bool(wanted >> i & 1)) for i, v in enumerate((x, w, b))]
        ops.layer_norm(*t).backward(dy)
        for i in range(3):
            assert (t[i].grad is None) if not wanted >> i & 1 else torch.equal(t[i].grad, want[i])
    a, c = x.clone().requires_grad_(True), b.clone().requires_grad_(True)
    ops.layer_norm(a, None, c).backward(dy)  # a bias alone
    assert torch.equal(a.grad, plain[0]) and torch.equal(c.grad, want[2])
    a = x.clone().requires_grad_(True)
    ops.layer_norm(a).backward(dy)
    assert torch.equal(a.grad, plain[0])


def test_node_refuses_tangents_and_changed_inputs():
    import torch.autograd.forward_ad as fw

    from synthefy_nori_b200 import ops

    x, w = torch.randn(4, 16, device="cuda"), torch.randn(16, device="cuda", requires_grad=True)
    with fw.dual_level(), pytest.raises(RuntimeError):
        ops.layer_norm(fw.make_dual(x, x), w)
    a = x.clone().requires_grad_(True)
    h = a * 1.0
    y = ops.layer_norm(h, w)
    h.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_node_in_a_captured_step():
    """Forward and backward captured and replayed on new values (with no eager graph of the leaf alive,
    whose accumulation node would tie autograd itself to the stream outside of the capture)."""
    from synthefy_nori_b200 import ops

    torch.manual_seed(4)
    x, w = torch.randn(60, 40, device="cuda"), torch.randn(40, device="cuda", requires_grad=True)
    dy = torch.randn(60, 40, device="cuda")

    def step():
        return torch.autograd.grad(ops.layer_norm(x, w), w, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.mul_(-1.5)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)

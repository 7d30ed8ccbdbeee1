"""LayerNorm forward and backward against the formulas in 64 bits.

Tolerances.  A row's mean is a sum of at most 32 values a thread and 8 + 5 pairwise steps, its
variance the same over squares: with u = 2^-24 every normalised value is within
64 u (max|x| rstd + |xhat|) of the exact one.  dx sums as many products of such values.  The
weight's sums add at most 8 rows a thread in these tests, then 32 row groups, 37 + 8 partial
rows: 128 u of the sum of magnitudes, and 64 u max|x| rstd of each xhat.  The results' own
roundings (half a step of the type) come on top."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


def ln64(x, w, b, eps=EPS):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = (x.var(-1, unbiased=False, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    y = h * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    return y, h, mean, rstd


def check(x, w, b, dy, out_dtype, ops, rows_view=None):
    y64, h, mean64, rstd64 = ln64(x, w, b)
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, EPS, out_dtype)
    assert y.dtype == (out_dtype or x.dtype) and y.shape == x.shape and y.is_contiguous()
    amp = x.double().abs().amax(-1, keepdim=True) * rstd64  # max|x| rstd of each row
    wmax = 1.0 if w is None else w.double().abs()
    herr = 64 * U * (amp + h.abs())
    half = lambda t: torch.finfo(t.dtype).eps / 2  # noqa: E731
    assert ((y.double() - y64).abs() <= herr * wmax + half(y) * y64.abs() + 4 * U * y64.abs() + 1e-7 * (y.dtype == torch.float16)).all()
    assert ((mean.double() - mean64.flatten()).abs() <= 64 * U * x.double().abs().amax(-1).flatten()).all()
    assert ((rstd.double() / rstd64.flatten() - 1).abs() <= 128 * U * (1 + amp.flatten() ** 2)).all()

    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w, weight_grad=True, bias_grad=True)
    assert dx.dtype == x.dtype and dx.shape == x.shape and dw.dtype == db.dtype == torch.float32
    d = dy.double()
    q = d * (1.0 if w is None else w.double())
    dx64 = rstd64 * (q - q.mean(-1, keepdim=True) - h * (q * h).mean(-1, keepdim=True))
    qmax, hmax = q.abs().amax(-1, keepdim=True), h.abs().amax(-1, keepdim=True)
    # q, mean(q), h mean(q h): each with its own error and that of h and rstd
    err = rstd64 * qmax * (8 * U + (1 + hmax) * (64 * U * (1 + hmax) + 2 * 64 * U * (amp + hmax)) + 256 * U * (1 + amp ** 2))
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0  # half a step of fp16's subnormal range
    assert ((dx.double() - dx64).abs() <= err + half(dx) * dx64.abs() + sub).all()
    cols = lambda t: t.reshape(-1, x.shape[-1]).sum(0)  # noqa: E731
    dw_err = d.abs() * (h.abs() * 128 * U + 64 * U * (amp + h.abs()) + 128 * U * (1 + amp ** 2) * h.abs())
    assert ((dw.double() - cols(d * h)).abs() <= cols(dw_err) + 1e-30).all()
    assert ((db.double() - cols(d)).abs() <= 128 * U * cols(d.abs()) + 1e-30).all()
    return y, dx, dw, db


@pytest.mark.parametrize("tx,ty", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (37, 64), (5, 8), (1000, 60), (333, 127), (64, 256), (17, 258),
                                       (100, 448), (9, 999), (40, 1024), (3, 1344), (6, 2050), (2, 4096), (5, 8192),
                                       (4, 8193), (70, 9000), (1, 20000)])
def test_forward_backward(rows, cols, tx, ty):
    from synthefy_nori_b200 import ops

    torch.manual_seed(rows + cols)
    x = (torch.randn(rows, cols, device="cuda") * 2 + torch.randn(rows, 1, device="cuda")).to(tx)
    w, b = 1 + 0.3 * torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    dy = torch.randn(rows, cols, device="cuda").to(ty)
    if cols == 1:  # one column: xhat is 0 and so is dx
        y, mean, rstd = ops.layer_norm_fwd(x, w, b, EPS, ty)
        torch.testing.assert_close(y, b.to(ty).expand(rows, 1))
        dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
        assert (dx == 0).all() and (dw == 0).all()
        return
    out = torch.float32 if ty != tx else None
    first = check(x, w, b, dy, out, ops)
    again = check(x, w, b, dy, out, ops)
    assert all(torch.equal(s, t) for s, t in zip(first, again))  # fixed order of the sums
    check(x, None, None, dy, out, ops)


def test_many_rows():
    """More rows than a grid holds at once."""
    from synthefy_nori_b200 import ops

    torch.manual_seed(0)
    x = torch.randn(18000, 72, device="cuda").to(torch.bfloat16)
    check(x, torch.randn(72, device="cuda"), None, torch.randn_like(x), None, ops)


def test_strides_and_shapes():
    from synthefy_nori_b200 import ops

    torch.manual_seed(1)
    base = torch.randn(6, 5, 3, 100, device="cuda")
    w, b = torch.randn(64, device="cuda"), torch.randn(64, device="cuda")
    for x in (base[..., 7:71], base[:, :, 0, 8:72], base[::2, 1:4, :, :64], base[0, 0, 0, 4:68],
              base.transpose(0, 3)[:64, :, :, :].permute(1, 2, 3, 0), base[:1, :, :1, :64].expand(4, 5, 2, 64)):
        dy = torch.randn(x.shape, device="cuda")
        check(x, w, b, dy, None, ops)
        check(x.to(torch.bfloat16), w, b, dy, torch.float32, ops)
    # a weight that starts off a 16-byte boundary, and a gradient with strided rows
    wv = torch.randn(65, device="cuda")[1:]
    x = torch.randn(33, 64, device="cuda")
    check(x, wv, b, torch.randn(33, 200, device="cuda")[:, 9:73], None, ops)
    y, mean, rstd = ops.layer_norm_fwd(x[:0], w, b)
    assert y.shape == (0, 64)
    dx, dw, db = ops.layer_norm_bwd(x[:0], x[:0], mean, rstd, w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_unwanted_gradients():
    from synthefy_nori_b200 import ops

    torch.manual_seed(2)
    for C in (48, 700, 5000, 9000):
        x, dy, w = (torch.randn(50, C, device="cuda"), torch.randn(50, C, device="cuda"), torch.randn(C, device="cuda"))
        _, mean, rstd = ops.layer_norm_fwd(x, w)
        full = ops.layer_norm_bwd(dy, x, mean, rstd, w)
        for wg in (False, True):
            for bg in (False, True):
                part = ops.layer_norm_bwd(dy, x, mean, rstd, w, weight_grad=wg, bias_grad=bg)
                assert torch.equal(part[0], full[0])
                assert (part[1] is None) != wg and (part[2] is None) != bg
                assert not wg or torch.equal(part[1], full[1])
                assert not bg or torch.equal(part[2], full[2])


def test_constant_and_extreme_rows():
    from synthefy_nori_b200 import ops

    C = 96
    x = torch.stack([torch.full((C,), 3.0), torch.zeros(C), torch.linspace(-1, 1, C) * 1e15, torch.linspace(-1, 1, C) * 1e-20,
                     torch.linspace(0, 1, C) + 4096.0, torch.full((C,), float("nan")), torch.linspace(-1, 1, C)]).cuda()
    x[6, 5] = float("inf")
    w, b = torch.full((C,), 2.0, device="cuda"), torch.full((C,), 0.5, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, EPS)
    assert torch.equal(y[:2], torch.full((2, C), 0.5, device="cuda"))  # no variance: the bias alone
    ref = ln64(x[:5], w, b)[0]
    # row 4: its mean is 4096 in a range of 1: the mean's rounding is 64 u 4097 rstd
    assert ((y[:5].double() - ref).abs().amax(1) <= 2 * 64 * U * torch.tensor([1, 1, 4, 4, 4097 / 0.29], device="cuda") + 1e-6).all()
    assert y[5].isnan().all() and y[6].isnan().any() and y[:5].isfinite().all()


@pytest.mark.parametrize("tx,out", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32)])
def test_autograd(tx, out):
    from synthefy_nori_b200 import ops

    torch.manual_seed(3)
    x = torch.randn(4, 9, 80, device="cuda").to(tx).requires_grad_(True)
    w = torch.nn.Parameter(1 + 0.2 * torch.randn(80, device="cuda"))
    b = torch.nn.Parameter(torch.randn(80, device="cuda"))
    y = ops.layer_norm(x, w, b, out_dtype=out)
    c = torch.randn(y.shape, device="cuda").to(y.dtype)
    got = torch.autograd.grad((y * c).sum(), (x, w, b))
    xd, wd, bd = (t.detach().double().requires_grad_(True) for t in (x, w, b))
    want = torch.autograd.grad((torch.nn.functional.layer_norm(xd, (80,), wd, bd) * c.double()).sum(), (xd, wd, bd))
    for g, r, t in zip(got, want, (x, w, b)):
        assert g.dtype == t.dtype and g.shape == t.shape
        # dy is exact; each value is within 2^-17 of the largest and half a step of its type
        assert ((g.double() - r).abs() <= 2.0 ** -17 * r.abs().amax() + torch.finfo(g.dtype).eps / 2 * r.abs()).all()
    # gradients of the weight alone, of the input alone
    y = ops.layer_norm(x.detach(), w, None, out_dtype=out)
    assert torch.autograd.grad((y * c).sum(), w)[0].shape == (80,)
    y = ops.layer_norm(x, w.detach(), b.detach(), out_dtype=out)
    assert torch.equal(torch.autograd.grad((y * c).sum(), x)[0], got[0])


def test_gradient_against_differences():
    from synthefy_nori_b200 import ops

    torch.manual_seed(4)
    x = torch.randn(3, 20, device="cuda", requires_grad=True)
    w = torch.randn(20, device="cuda", requires_grad=True)
    b = torch.randn(20, device="cuda", requires_grad=True)
    c = torch.randn(3, 20, device="cuda")
    f = lambda *t: float((ops.layer_norm(*t).double() * c).sum())  # noqa: E731
    grads = torch.autograd.grad((ops.layer_norm(x, w, b) * c).sum(), (x, w, b))
    h = 2.0 ** -7  # truncation h^2/6 of a third derivative of order 10, rounding 60 * 2^-22 / h
    for k, (t, g) in enumerate(zip((x, w, b), grads)):
        for i in range(0, t.numel(), 7):
            e = torch.zeros_like(t).view(-1)
            e[i] = h
            args = [x.detach(), w.detach(), b.detach()]
            up, dn = list(args), list(args)
            up[k], dn[k] = args[k] + e.view(t.shape), args[k] - e.view(t.shape)
            assert abs((f(*up) - f(*dn)) / (2 * h) - float(g.view(-1)[i])) < 10 * h * h / 6 * 10 + 60 * 2.0 ** -22 / h


@pytest.mark.parametrize("shape", [(3, 16), (2, 3, 16), (16,)])
def test_second_derivative(shape):
    from synthefy_nori_b200 import ops

    torch.manual_seed(5)
    x = torch.randn(*shape, device="cuda", requires_grad=True)
    w = torch.randn(16, device="cuda", requires_grad=True)
    c = torch.randn(*shape, device="cuda")

    def penalty(fn, xx, ww, cc):
        g, gw = torch.autograd.grad((fn(xx, ww).square() * cc).sum(), (xx, ww), create_graph=True)
        return torch.autograd.grad(g.square().sum() + gw.square().sum(), (xx, ww))

    got = penalty(lambda a, v: ops.layer_norm(a, v), x, w, c)
    xd, wd = (t.detach().double().requires_grad_(True) for t in (x, w))
    want = penalty(lambda a, v: torch.nn.functional.layer_norm(a, (16,), v), xd, wd, c.double())
    for g, r in zip(got, want):
        assert float((g.double() - r).norm() / r.norm()) < 1e-5


def test_graph_replay_and_streams():
    from synthefy_nori_b200 import ops

    torch.manual_seed(6)
    x = torch.randn(700, 448, device="cuda").to(torch.bfloat16)
    dy, w = torch.randn_like(x), torch.randn(448, device="cuda")

    def step():
        y, mean, rstd = ops.layer_norm_fwd(x, w)
        return (y, *ops.layer_norm_bwd(dy, x, mean, rstd, w))

    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.mul_(-1)  # replay reads the inputs anew
    want = [t.clone() for t in step()]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_model_modules_run_the_kernel():
    """LayerNorm modules of the model: parameters of the same names, results of torch's."""
    from synthefy_nori_b200.models.layers import LayerNorm, LayerNormMixedPrecision

    torch.manual_seed(7)
    for cls, affine in ((LayerNorm, True), (LayerNormMixedPrecision, True), (LayerNormMixedPrecision, False)):
        m = cls(72, elementwise_affine=affine).cuda()
        t = torch.nn.LayerNorm(72, elementwise_affine=affine).cuda()
        assert list(m.state_dict()) == list(t.state_dict())
        if affine:
            torch.nn.init.normal_(m.weight)
            t.load_state_dict(m.state_dict())
        x = torch.randn(2, 5, 72, device="cuda")
        torch.testing.assert_close(m(x), t(x), atol=2e-6, rtol=2e-6)
        for dt in (torch.bfloat16, torch.float16):
            with torch.autocast("cuda", dtype=dt):
                y, r = m(x.to(dt)), t(x.to(dt))
            want = torch.float16 if cls is LayerNormMixedPrecision and dt == torch.float16 else torch.float32
            assert y.dtype == want
            torch.testing.assert_close(y.float(), r, atol=2e-3 if want != torch.float32 else 2e-6, rtol=2e-3 if want != torch.float32 else 2e-6)


def test_refusals():
    from synthefy_nori_b200 import ops

    x = torch.randn(4, 16, device="cuda")
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x.double())
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, out_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.layer_norm_fwd(x, torch.ones(15, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.layer_norm_fwd(x, torch.ones(16))
    with pytest.raises(RuntimeError):
        ops.layer_norm_fwd(x, eps=-1.0)
    with pytest.raises(RuntimeError):
        ops.layer_norm_fwd(x[:, :0])
    _, mean, rstd = ops.layer_norm_fwd(x)
    with pytest.raises(RuntimeError):
        ops.layer_norm_bwd(x[:3], x, mean, rstd)
    with pytest.raises(RuntimeError):
        ops.layer_norm_bwd(x.to(torch.bfloat16), x, mean, rstd)
    with pytest.raises(RuntimeError):
        ops.layer_norm_bwd(x, x, mean[:3], rstd)

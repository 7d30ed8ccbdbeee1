"""After a bounded wait has run out (the status word is set) the tcgen05 kernels return without a result, and
work again once it is cleared."""

import pytest
import torch

pytestmark = pytest.mark.gpu

H, D, B, T, N = 2, 56, 2, 5, 300


def _calls():
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    A = H * D
    y, do = rnd(B * N * T, 3 * A), rnd(B * N * T, A)
    q, k, v = y[:, :A], y[:, A : 2 * A], y[:, 2 * A :]
    seq = lambda w: (N * T * w, w, D, T * w, T, H)  # noqa: E731
    feat = lambda w: (T * w, 0, D, w, 1, H)  # noqa: E731
    s3, s1, f3, f1 = seq(3 * A), seq(A), feat(3 * A), feat(A)
    o_seq, o_feat = torch.empty_like(do), torch.empty_like(do)
    lse_seq = torch.empty(B * T * H, N, device="cuda")
    lse_feat = torch.empty(B * N * H, T, device="cuda")
    kw_s, kw_f = dict(BH=B * T * H, Nq=N, Nk=N, d=D, scale=D ** -0.5), dict(BH=B * N * H, T=T, d=D, scale=D ** -0.5)
    ops.attention_fwd_tc(q, k, v, o_seq, lq=s3, lk=s3, lv=s3, lo=s1, lse=lse_seq, **kw_s)
    ops.attention_feat_fwd_tc(q, k, v, o_feat, lq=f3, lk=f3, lv=f3, lo=f1, lse=lse_feat, **kw_f)
    a, w, x = rnd(700, 192), rnd(320, 192), rnd(700, 320)
    return {
        "gemm": (lambda r: ops.gemm(a, w, out=r[0]), [torch.empty(700, 320, device="cuda", dtype=torch.bfloat16)]),
        "gemm_residual": (lambda r: ops.gemm_residual(a, w, x, 0.5, out=r[0]), [torch.empty_like(x)]),
        "attention": (lambda r: ops.attention_fwd_tc(q, k, v, r[0], lq=s3, lk=s3, lv=s3, lo=s1, lse=r[1], **kw_s),
                      [torch.empty_like(do), torch.empty_like(lse_seq)]),
        "attention_bwd": (lambda r: ops.attention_bwd_tc(q, k, v, o_seq, do, lse_seq, r[0], r[1], r[2], lq=s3, lkv=s3, lo=s1,
                                                         ldo=s1, ldkv=s1, ldq=s1, **kw_s),
                          [torch.zeros(B * N * T, A, device="cuda"), torch.empty_like(do), torch.empty_like(do)]),
        "feature_attention": (lambda r: ops.attention_feat_fwd_tc(q, k, v, r[0], lq=f3, lk=f3, lv=f3, lo=f1, lse=r[1], **kw_f),
                              [torch.empty_like(do), torch.empty_like(lse_feat)]),
        "feature_attention_bwd": (lambda r: ops.attention_feat_bwd_tc(q, k, v, o_feat, do, lse_feat, r[0], r[1], r[2], lq=f3,
                                                                      lkv=f3, lo=f1, lg=f1, **kw_f),
                                  [torch.empty_like(do) for _ in "qkv"]),
    }


@pytest.mark.parametrize("name", ["gemm", "gemm_residual", "attention", "attention_bwd", "feature_attention",
                                  "feature_attention_bwd"])
def test_nothing_is_written_after_a_timeout(name):
    from synthefy_nori_b200 import ops

    call, res = _calls()[name]
    call(res)
    want = [t.clone() for t in res]
    word = ops.status_word(res[0].device)
    fill = 0.0 if name == "attention_bwd" else 7.0  # (its first result is an accumulator)
    for t in res:
        t.fill_(fill)
    try:
        word.fill_(2)
        for _ in range(3):
            call(res)
        with pytest.raises(RuntimeError, match="timeout"):
            ops.check_status(res[0].device)
    finally:
        word.zero_()
    assert all((t == fill).all() for t in res)
    call(res)
    for t, w in zip(res, want):
        assert torch.equal(t, w) if name != "attention_bwd" else torch.allclose(t, w, rtol=1e-2, atol=1e-2)

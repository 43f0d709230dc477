"""CPU checks of the 8-bit and grouped-router entry points: what the C ABI
refuses, before anything is launched."""

import ctypes as C

import pytest

from table_moe import _native as N

P = C.c_void_p(1 << 12)   # aligned, never read: every call below is refused or empty
ODD = C.c_void_p((1 << 12) + 8)


@pytest.fixture(scope="module")
def lib():
    return N.load()


def _route(lib, dtype=N.TM_DT_F32, logits=P, n=4, e=64, ld=64, bias=None, scoring=0, groups=1, keep=1, rule=0, k=4,
           norm=0, scale=1.0, w=P, i=P):
    return lib.tm_route_experts(dtype, logits, n, e, ld, bias, scoring, groups, keep, rule, k, norm, scale, w, i, None)


def test_route_experts_refusals(lib):
    assert _route(lib, n=0) == N.TM_OK
    assert _route(lib, n=0, logits=None) == N.TM_OK
    for kw, want in ((dict(dtype=7), N.TM_EINVAL_DTYPE), (dict(dtype=3), N.TM_EINVAL_DTYPE),
                     (dict(e=0), N.TM_EINVAL_SHAPE), (dict(e=1025, ld=1025), N.TM_EINVAL_SHAPE),
                     (dict(ld=63), N.TM_EINVAL_SHAPE), (dict(n=-1), N.TM_EINVAL_SHAPE),
                     (dict(scoring=2), N.TM_EINVAL_ARG), (dict(rule=-1), N.TM_EINVAL_ARG),
                     (dict(groups=5), N.TM_EINVAL_SHAPE), (dict(groups=0), N.TM_EINVAL_SHAPE),
                     (dict(groups=8, keep=9), N.TM_EINVAL_SHAPE), (dict(groups=8, keep=0), N.TM_EINVAL_SHAPE),
                     (dict(groups=8, keep=1, k=9), N.TM_EINVAL_SHAPE), (dict(k=0), N.TM_EINVAL_SHAPE),
                     (dict(k=33), N.TM_EINVAL_SHAPE), (dict(e=512, ld=512, groups=128), N.TM_EINVAL_SHAPE),
                     (dict(scale=float("nan")), N.TM_EINVAL_ARG), (dict(logits=None), N.TM_EINVAL_ARG),
                     (dict(w=None), N.TM_EINVAL_ARG), (dict(i=None), N.TM_EINVAL_ARG)):
        assert _route(lib, **kw) == want, kw


def test_quantiser_refusals(lib):
    rows = lambda dtype=N.TM_DT_BF16, x=P, n=4, k=200, ld=200, q=P, ldq=256, s=P, lds=2: lib.tm_fp8_quantize_rows(  # noqa: E731
        dtype, x, n, k, ld, q, ldq, s, lds, None)
    assert rows(n=0, x=None) == N.TM_OK
    for kw, want in ((dict(dtype=3), N.TM_EINVAL_DTYPE), (dict(k=0, ld=0), N.TM_EINVAL_SHAPE),
                     (dict(ld=199), N.TM_EINVAL_SHAPE), (dict(ldq=200), N.TM_EINVAL_SHAPE),
                     (dict(ldq=264), N.TM_EINVAL_SHAPE), (dict(lds=1), N.TM_EINVAL_SHAPE),
                     (dict(n=-1), N.TM_EINVAL_SHAPE), (dict(x=None), N.TM_EINVAL_ARG), (dict(q=None), N.TM_EINVAL_ARG),
                     (dict(s=None), N.TM_EINVAL_ARG), (dict(q=ODD), N.TM_EINVAL_SHAPE),
                     (dict(n=1 << 40), N.TM_EINVAL_SHAPE)):
        assert rows(**kw) == want, kw
    wt = lambda dtype=N.TM_DT_BF16, w=P, m=2, n=130, k=200, q=P, ldq=256, s=P: lib.tm_fp8_quantize_weight(  # noqa: E731
        dtype, w, m, n, k, q, ldq, s, None)
    assert wt(m=0, w=None) == N.TM_OK
    for kw, want in ((dict(dtype=9), N.TM_EINVAL_DTYPE), (dict(m=-1), N.TM_EINVAL_SHAPE), (dict(n=0), N.TM_EINVAL_SHAPE),
                     (dict(k=0), N.TM_EINVAL_SHAPE), (dict(ldq=200), N.TM_EINVAL_SHAPE), (dict(w=None), N.TM_EINVAL_ARG),
                     (dict(q=None), N.TM_EINVAL_ARG), (dict(s=None), N.TM_EINVAL_ARG), (dict(q=ODD), N.TM_EINVAL_SHAPE),
                     (dict(m=1 << 30), N.TM_EINVAL_SHAPE)):
        assert wt(**kw) == want, kw


def test_linear_refusals(lib):
    need = lib.tm_fp8_linear_workspace_size(4, 256, N.TM_DT_BF16)
    assert need >= 4 * 256 and lib.tm_fp8_linear_workspace_size(0, 256, N.TM_DT_BF16) == 0

    def f(dtype=N.TM_DT_BF16, x=P, xs=None, n=4, k=256, ldx=256, ldxs=0, w=P, ws=P, out_n=64, bias=None, y=P, ldy=64,
          wk=P, nb=None):
        return lib.tm_fp8_linear(dtype, x, xs, n, k, ldx, ldxs, w, ws, out_n, bias, y, ldy, wk,
                                 need if nb is None else nb, None)

    assert f(n=0, x=None) == N.TM_OK
    for kw, want in ((dict(dtype=3), N.TM_EINVAL_DTYPE), (dict(k=0), N.TM_EINVAL_SHAPE),
                     (dict(k=16385, ldx=16385), N.TM_EINVAL_SHAPE), (dict(n=-1), N.TM_EINVAL_SHAPE),
                     (dict(out_n=0), N.TM_EINVAL_SHAPE), (dict(ldx=255), N.TM_EINVAL_SHAPE),
                     (dict(ldy=63), N.TM_EINVAL_SHAPE), (dict(xs=P, ldx=255, ldxs=2), N.TM_EINVAL_SHAPE),
                     (dict(xs=P, ldxs=1), N.TM_EINVAL_SHAPE), (dict(xs=P, ldxs=2, x=ODD), N.TM_EINVAL_SHAPE),
                     (dict(x=None), N.TM_EINVAL_ARG), (dict(w=None), N.TM_EINVAL_ARG), (dict(ws=None), N.TM_EINVAL_ARG),
                     (dict(y=None), N.TM_EINVAL_ARG), (dict(w=ODD), N.TM_EINVAL_SHAPE),
                     (dict(wk=None), N.TM_EWORKSPACE), (dict(nb=need - 1), N.TM_EWORKSPACE),
                     (dict(wk=ODD), N.TM_EWORKSPACE)):
        assert f(**kw) == want, kw


def _experts(e=4, h=256, inter=128, w=1 << 12, s=1 << 12):
    return N.Fp8Experts(e, h, inter, 0, w, s, w, s, w, s)


def test_expert_refusals(lib):
    ex = _experts()
    need = lib.tm_fp8_grouped_swiglu_workspace_size(C.byref(ex), 8, 2)
    assert need > 0
    assert lib.tm_fp8_grouped_swiglu_workspace_size(C.byref(ex), 0, 2) == 0
    assert lib.tm_fp8_grouped_swiglu_workspace_size(None, 8, 2) == 0
    # never less for more tokens
    sizes = [lib.tm_fp8_grouped_swiglu_workspace_size(C.byref(ex), n, 2) for n in range(1, 700, 7)]
    assert sizes == sorted(sizes)

    def f(ex=ex, dtype=N.TM_DT_BF16, x=P, n=8, ldx=256, ids=P, k=2, ldi=2, mask=P, out=P, so_b=512, so_s=256, ws=P,
          nb=None):
        return lib.tm_fp8_grouped_swiglu(None if ex is None else C.byref(ex), dtype, x, n, ldx, ids, k, ldi, mask, 1, 0,
                                         out, so_b, so_s, ws, need if nb is None else nb, None)

    assert f(n=0, x=None) == N.TM_OK
    for kw, want in ((dict(ex=None), N.TM_EINVAL_ARG), (dict(dtype=N.TM_DT_F32), N.TM_EINVAL_DTYPE),
                     (dict(ex=_experts(h=200)), N.TM_EINVAL_SHAPE), (dict(ex=_experts(inter=64)), N.TM_EINVAL_SHAPE),
                     (dict(ex=_experts(e=0)), N.TM_EINVAL_SHAPE), (dict(ex=_experts(e=1025)), N.TM_EINVAL_SHAPE),
                     (dict(ex=_experts(h=16512)), N.TM_EINVAL_SHAPE), (dict(ex=_experts(w=None)), N.TM_EINVAL_ARG),
                     (dict(ex=_experts(s=None)), N.TM_EINVAL_ARG), (dict(ex=_experts(w=24)), N.TM_EINVAL_SHAPE),
                     (dict(n=-1), N.TM_EINVAL_SHAPE), (dict(k=0), N.TM_EINVAL_SHAPE), (dict(ldi=1), N.TM_EINVAL_SHAPE),
                     (dict(ldx=255), N.TM_EINVAL_SHAPE), (dict(ldx=257), N.TM_EINVAL_SHAPE),
                     (dict(x=ODD), N.TM_EINVAL_SHAPE), (dict(out=ODD), N.TM_EINVAL_SHAPE),
                     (dict(so_b=516), N.TM_EINVAL_SHAPE), (dict(so_s=4), N.TM_EINVAL_SHAPE),
                     (dict(x=None), N.TM_EINVAL_ARG), (dict(ids=None), N.TM_EINVAL_ARG),
                     (dict(mask=None), N.TM_EINVAL_ARG), (dict(out=None), N.TM_EINVAL_ARG),
                     (dict(ws=None), N.TM_EWORKSPACE), (dict(nb=need - 1), N.TM_EWORKSPACE),
                     (dict(ws=ODD), N.TM_EWORKSPACE)):
        assert f(**kw) == want, kw

    one = _experts(e=1)
    need1 = lib.tm_fp8_expert_swiglu_workspace_size(C.byref(one), 8)
    assert need1 > 0 and lib.tm_fp8_expert_swiglu_workspace_size(C.byref(one), 0) == 0

    def g(ex=one, dtype=N.TM_DT_F16, x=P, n=8, ldx=256, add=None, lda=256, out=P, ldo=256, ws=P, nb=None):
        return lib.tm_fp8_expert_swiglu(C.byref(ex), dtype, x, n, ldx, add, lda, out, ldo, ws,
                                        need1 if nb is None else nb, None)

    assert g(n=0, x=None) == N.TM_OK
    for kw, want in ((dict(ex=_experts(e=2)), N.TM_EINVAL_SHAPE), (dict(dtype=N.TM_DT_F32), N.TM_EINVAL_DTYPE),
                     (dict(ldx=128), N.TM_EINVAL_SHAPE), (dict(ldo=128), N.TM_EINVAL_SHAPE),
                     (dict(add=P, lda=128), N.TM_EINVAL_SHAPE), (dict(add=ODD), N.TM_EINVAL_SHAPE),
                     (dict(x=None), N.TM_EINVAL_ARG), (dict(out=None), N.TM_EINVAL_ARG),
                     (dict(nb=need1 - 1), N.TM_EWORKSPACE), (dict(ws=None), N.TM_EWORKSPACE)):
        assert g(**kw) == want, kw


def test_host_tensors_are_refused():
    import torch

    from table_moe.ops import Fp8GroupedExperts, Fp8Linear, quantize_rows_fp8, quantize_weight_fp8, route_experts

    x = torch.zeros(4, 128)
    with pytest.raises(RuntimeError):
        quantize_rows_fp8(x)
    with pytest.raises(RuntimeError):
        quantize_weight_fp8(x)
    with pytest.raises(RuntimeError):
        route_experts(x, 2)
    q, s = torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.ones(1, 1)
    with pytest.raises(RuntimeError):
        Fp8Linear(q, s)
    with pytest.raises(RuntimeError):
        Fp8GroupedExperts(*(3 * [q[None], s[None]]))


def test_route_experts_refuses_an_infinite_scale(lib):
    """0 * inf is NaN: an expert that is not available has weight 0."""
    for scale in (float("inf"), float("-inf"), float("nan")):
        assert _route(lib, scale=scale, n=0) == N.TM_EINVAL_ARG
    assert _route(lib, scale=-3.0e38, n=0) == N.TM_OK


def test_quantise_rows_refuses_counts_past_64_bits(lib):
    """n_rows times a row's blocks out of int64's range."""
    for n, k in ((1 << 61, 1024), ((1 << 61) + 16, 1024), ((1 << 63) - 1, 129), (1 << 60, 1 << 20)):
        assert lib.tm_fp8_quantize_rows(N.TM_DT_BF16, P, n, k, k, P, -(-k // 128) * 128, P, -(-k // 128),
                                        None) == N.TM_EINVAL_SHAPE, (n, k)

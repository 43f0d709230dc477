"""CPU checks of the rotation's and the 8-bit cache's entry points: what the C
ABI refuses, before anything is launched."""

import ctypes as C

import pytest

from table_moe import _native as N

P = C.c_void_p(1 << 12)   # aligned, never read: every call below is refused or empty
ODD = C.c_void_p((1 << 12) + 8)


@pytest.fixture(scope="module")
def lib():
    return N.load()


def test_rotate_refusals(lib):
    def f(dtype=N.TM_DT_BF16, q=P, n=4, h=2, k=P, hk=1, d=128, r=128, pos=P, ldp=4, sec=(24, 20, 20), inv=P, qo=P, ko=P):
        return lib.tm_rotate_positions(dtype, q, n, h, 256, 128, k, hk, 128, 128, d, r, pos, ldp, len(sec),
                                       (C.c_int32 * len(sec))(*sec) if sec else None, 1, 0, 0, inv, qo, 256, 128, ko,
                                       128, 128, None)

    assert f(n=0, q=None, pos=None, inv=None, qo=None) == N.TM_OK
    for kw, want in ((dict(dtype=3), N.TM_EINVAL_DTYPE), (dict(n=-1), N.TM_EINVAL_SHAPE), (dict(h=0), N.TM_EINVAL_SHAPE),
                     (dict(hk=0), N.TM_EINVAL_SHAPE), (dict(d=0), N.TM_EINVAL_SHAPE), (dict(d=1025), N.TM_EINVAL_SHAPE),
                     (dict(r=127), N.TM_EINVAL_SHAPE), (dict(r=130), N.TM_EINVAL_SHAPE), (dict(r=0), N.TM_EINVAL_SHAPE),
                     (dict(ldp=3), N.TM_EINVAL_SHAPE), (dict(sec=()), N.TM_EINVAL_SHAPE),
                     (dict(sec=(10, 10, 10, 10, 24)), N.TM_EINVAL_SHAPE), (dict(sec=(24, 20, 21)), N.TM_EINVAL_SHAPE),
                     (dict(sec=(-4, 48, 20)), N.TM_EINVAL_SHAPE), (dict(sec=(2 ** 31 - 1, 2 ** 31 - 1, 66)), N.TM_EINVAL_SHAPE),
                     (dict(q=None), N.TM_EINVAL_ARG), (dict(pos=None), N.TM_EINVAL_ARG), (dict(inv=None), N.TM_EINVAL_ARG),
                     (dict(qo=None), N.TM_EINVAL_ARG), (dict(ko=None), N.TM_EINVAL_ARG)):
        assert f(**kw) == want, kw


def _cache(pages=8, heads=2, d=128, dv=128, page=64, k=1 << 12, v=1 << 12, ks=1 << 12, vs=1 << 12):
    return N.Kv8Cache(pages, heads, d, dv, page, k, v, ks, vs)


def _batch(table=1 << 12, ld=4, lengths=1 << 12, starts=None, seqs=3, tokens=3, most=4):
    return N.Kv8Batch(table, ld, lengths, starts, seqs, tokens, most, 0)


BAD_CACHE = [dict(pages=-1), dict(pages=1 << 31), dict(heads=0), dict(heads=1025), dict(page=16), dict(page=96),
             dict(d=96), dict(d=64), dict(dv=192), dict(d=0)]
BAD_BATCH = [dict(seqs=-1), dict(tokens=-1), dict(tokens=4), dict(most=-1), dict(ld=3), dict(seqs=1 << 24, tokens=1 << 24)]


def _refused_descriptions(call):
    for kw in BAD_CACHE:
        assert call(c=_cache(**kw)) == N.TM_EINVAL_SHAPE, kw
    for kw in BAD_BATCH:
        assert call(b=_batch(**kw)) == N.TM_EINVAL_SHAPE, kw
    for kw in (dict(k=None), dict(v=None), dict(ks=None), dict(vs=None)):
        assert call(c=_cache(**kw)) == N.TM_EINVAL_ARG, kw
    for kw in (dict(table=None), dict(lengths=None)):
        assert call(b=_batch(**kw)) == N.TM_EINVAL_ARG, kw
    assert call(c=_cache(k=(1 << 12) + 8)) == N.TM_EINVAL_SHAPE
    assert call(c=None) == N.TM_EINVAL_ARG and call(b=None) == N.TM_EINVAL_ARG
    assert call(b=_batch(seqs=0, tokens=0, lengths=None, table=None)) == N.TM_OK


def _ref(x):
    return None if x is None else C.byref(x)


def test_append_refusals(lib):
    def f(c=_cache(), b=_batch(), dtype=N.TM_DT_F32, k=P, kt=256, kh=128, v=P, vt=256, vh=128):
        return lib.tm_kv8_append(_ref(c), _ref(b), dtype, k, kt, kh, v, vt, vh, None)

    _refused_descriptions(f)
    assert f(b=_batch(most=0, table=None)) == N.TM_OK
    for kw, want in ((dict(dtype=3), N.TM_EINVAL_DTYPE), (dict(k=None), N.TM_EINVAL_ARG), (dict(v=None), N.TM_EINVAL_ARG),
                     (dict(k=ODD), N.TM_EINVAL_SHAPE), (dict(v=ODD), N.TM_EINVAL_SHAPE), (dict(kt=252), N.TM_EINVAL_SHAPE),
                     (dict(vh=4), N.TM_EINVAL_SHAPE)):
        assert f(**kw) == want, kw


def test_attention_refusals(lib):
    need = lib.tm_kv8_attention_workspace_size(C.byref(_cache()), C.byref(_batch(most=4096, ld=4096)), 4)
    assert need > 0

    def f(c=_cache(), b=_batch(most=4096, ld=4096), dtype=N.TM_DT_BF16, q=P, qt=512, qh=128, h=4, scale=0.1, out=P, ot=512,
          oh=128, ws=P, nb=need):
        return lib.tm_kv8_attention(_ref(c), _ref(b), dtype, q, qt, qh, h, scale, 1, out, ot, oh, None, ws, nb, None)

    _refused_descriptions(f)
    for kw, want in ((dict(dtype=N.TM_DT_F32), N.TM_EINVAL_DTYPE), (dict(h=3), N.TM_EINVAL_SHAPE), (dict(h=0), N.TM_EINVAL_SHAPE),
                     (dict(scale=0.0), N.TM_EINVAL_ARG), (dict(scale=-1.0), N.TM_EINVAL_ARG),
                     (dict(scale=float("nan")), N.TM_EINVAL_ARG), (dict(scale=float("inf")), N.TM_EINVAL_ARG),
                     (dict(q=None), N.TM_EINVAL_ARG), (dict(out=None), N.TM_EINVAL_ARG), (dict(q=ODD), N.TM_EINVAL_SHAPE),
                     (dict(out=ODD), N.TM_EINVAL_SHAPE), (dict(qt=516), N.TM_EINVAL_SHAPE), (dict(oh=4), N.TM_EINVAL_SHAPE),
                     (dict(ws=None), N.TM_EWORKSPACE), (dict(nb=need - 1), N.TM_EWORKSPACE), (dict(ws=ODD), N.TM_EWORKSPACE)):
        assert f(**kw) == want, kw
    assert lib.tm_kv8_attention_workspace_size(None, C.byref(_batch()), 4) == 0
    assert lib.tm_kv8_attention_workspace_size(C.byref(_cache()), C.byref(_batch(seqs=0, tokens=0)), 4) == 0


def test_importance_refusals(lib):
    need = lib.tm_kv8_importance_workspace_size(C.byref(_cache()), C.byref(_batch()), 4)
    assert need > 0

    def f(c=_cache(), b=_batch(), dtype=N.TM_DT_BF16, q=P, qt=512, qh=128, h=4, scale=0.1, lse=None, ldl=4, n=200, out=P,
          ldo=200, ws=P, nb=need):
        return lib.tm_kv8_importance(_ref(c), _ref(b), dtype, q, qt, qh, h, scale, lse, ldl, n, out, ldo, ws, nb, None)

    _refused_descriptions(f)
    assert f(n=0, out=None) == N.TM_OK
    for kw, want in ((dict(dtype=N.TM_DT_F32), N.TM_EINVAL_DTYPE), (dict(h=3), N.TM_EINVAL_SHAPE),
                     (dict(h=258), N.TM_EINVAL_SHAPE), (dict(scale=0.0), N.TM_EINVAL_ARG), (dict(n=-1), N.TM_EINVAL_SHAPE),
                     (dict(ldo=199), N.TM_EINVAL_SHAPE), (dict(lse=P, ldl=3), N.TM_EINVAL_SHAPE), (dict(q=None), N.TM_EINVAL_ARG),
                     (dict(out=None), N.TM_EINVAL_ARG), (dict(q=ODD), N.TM_EINVAL_SHAPE), (dict(qt=4), N.TM_EINVAL_SHAPE),
                     (dict(ws=None), N.TM_EWORKSPACE), (dict(nb=need - 1), N.TM_EWORKSPACE), (dict(ws=ODD), N.TM_EWORKSPACE)):
        assert f(**kw) == want, kw


def test_more_workgroups_than_a_launch_holds(lib):
    """2^24 workgroups of 256 threads are 2^32 threads: refused, not left to the runtime."""
    sections = (C.c_int32 * 1)(64)

    def rotate(n):
        return lib.tm_rotate_positions(N.TM_DT_BF16, P, n, 1, 128, 128, None, 0, 0, 0, 128, 128, P, n, 1, sections, 0, 0, 0,
                                       P, P, 128, 128, None, 0, 0, None)

    assert rotate(1 << 26) == N.TM_EINVAL_SHAPE and rotate((1 << 26) - 3) == N.TM_EINVAL_SHAPE
    assert rotate((1 << 31) - 1) == N.TM_EINVAL_SHAPE and rotate(1 << 31) == N.TM_EINVAL_SHAPE
    c = _cache(page=32)
    many = _batch(seqs=1 << 23, tokens=1 << 23, starts=1 << 12)
    assert lib.tm_kv8_append(C.byref(c), C.byref(many), N.TM_DT_BF16, P, 256, 128, P, 256, 128, None) == N.TM_EINVAL_SHAPE
    for seqs, tokens, starts in ((1 << 23, 1 << 23, None), (3, (1 << 28) - 8, 1 << 12), (3, 1 << 29, 1 << 12)):
        b = _batch(seqs=seqs, tokens=tokens, starts=starts)
        assert lib.tm_kv8_attention(C.byref(c), C.byref(b), N.TM_DT_BF16, P, 512, 128, 4, 0.1, 1, P, 512, 128, None, P,
                                    1 << 40, None) == N.TM_EINVAL_SHAPE, seqs

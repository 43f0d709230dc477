"""CPU checks of tm_kv8_importance_rows: what it refuses, before anything is launched."""

import ctypes as C

from table_moe import _native as N
from test_capi_kv8 import ODD, P, _batch, _cache, _ref, _refused_descriptions, lib  # noqa: F401


def test_importance_rows_refusals(lib):  # noqa: F811
    need = lib.tm_kv8_importance_workspace_size(C.byref(_cache()), C.byref(_batch()), 4)
    rows = _batch(starts=1 << 12, tokens=50)
    assert lib.tm_kv8_importance_workspace_size(C.byref(_cache()), C.byref(rows), 4) == need  # goes by the queries

    def f(c=_cache(), b=_batch(), dtype=N.TM_DT_BF16, q=P, qt=512, qh=128, h=4, scale=0.1, lse=None, ldl=4, out=P, ws=P,
          nb=need):
        return lib.tm_kv8_importance_rows(_ref(c), _ref(b), dtype, q, qt, qh, h, scale, lse, ldl, out, ws, nb, None)

    _refused_descriptions(f)
    assert f(b=_batch(starts=1 << 12, tokens=0), out=None, q=None) == N.TM_OK
    for b in (_batch(), rows):
        for kw, want in ((dict(dtype=N.TM_DT_F32), N.TM_EINVAL_DTYPE), (dict(h=3), N.TM_EINVAL_SHAPE),
                         (dict(h=258), N.TM_EINVAL_SHAPE), (dict(scale=0.0), N.TM_EINVAL_ARG),
                         (dict(lse=P, ldl=3), N.TM_EINVAL_SHAPE), (dict(q=None), N.TM_EINVAL_ARG),
                         (dict(out=None), N.TM_EINVAL_ARG), (dict(q=ODD), N.TM_EINVAL_SHAPE),
                         (dict(qt=4), N.TM_EINVAL_SHAPE), (dict(ws=None), N.TM_EWORKSPACE),
                         (dict(nb=need - 1), N.TM_EWORKSPACE), (dict(ws=ODD), N.TM_EWORKSPACE)):
            assert f(b=b, **kw) == want, kw

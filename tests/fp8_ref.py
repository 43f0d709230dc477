"""The 8-bit block format, the 8-bit expert MLP and the grouped router in
64 bits (numpy), written from their definitions: what the GPU tests compare
against.  Test infrastructure only."""

import numpy as np

BLOCK = 128
E4M3_MAX = 448.0


def e4m3_round(v):
    """Nearest e4m3 value (ties to even) of |v| <= 448; NaN stays NaN."""
    v = np.asarray(v, dtype=np.float64)
    a = np.abs(v)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.where(a > 0, a, 1.0)))
        e = np.where(np.ldexp(1.0, e.astype(int)) > a, e - 1, e)
        step = np.ldexp(1.0, (np.maximum(e, -6) - 3).astype(int))
        return np.sign(v) * np.rint(a / step) * step


def pow2_scale(amax):
    """Smallest power of two s >= 2^-126 with amax / s <= 448; 1 for 0."""
    amax = np.asarray(amax, dtype=np.float64)
    m, e = np.frexp(amax)
    p = np.maximum(e - 9 + (m > 0.875), -126)
    return np.where(amax > 0, np.ldexp(1.0, p), 1.0)


def _finite_max(x, axis):
    return np.where(np.isfinite(x), np.abs(x), 0.0).max(axis=axis)


def quantize_rows(x):
    """(q, scale) of x [M, K] in float64."""
    x = np.asarray(x, dtype=np.float64)
    m, k = x.shape
    kb = -(-k // BLOCK)
    b = np.zeros((m, kb * BLOCK))
    b[:, :k] = x
    b = b.reshape(m, kb, BLOCK)
    s = pow2_scale(_finite_max(b, 2))
    q = np.where(np.isfinite(b), b, np.nan) / s[:, :, None]
    return e4m3_round(q).reshape(m, -1)[:, :k], s


def quantize_weight(w):
    """(q, scale) of w [N, K] in float64."""
    w = np.asarray(w, dtype=np.float64)
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    b = np.zeros((nb * BLOCK, kb * BLOCK))
    b[:n, :k] = w
    b = b.reshape(nb, BLOCK, kb, BLOCK)
    s = pow2_scale(_finite_max(b, (1, 3)))
    q = np.where(np.isfinite(b), b, np.nan) / s[:, None, :, None]
    return e4m3_round(q).reshape(nb * BLOCK, -1)[:n, :k], s


def rows_value(q, s):
    return np.asarray(q, np.float64) * np.repeat(np.asarray(s, np.float64), BLOCK, 1)[:, :q.shape[1]]


def weight_value(q, s):
    n, k = q.shape
    s = np.repeat(np.repeat(np.asarray(s, np.float64), BLOCK, 0)[:n], BLOCK, 1)[:, :k]
    return np.asarray(q, np.float64) * s


def linear(x, wq, ws, bias=None):
    y = rows_value(*quantize_rows(x)) @ weight_value(wq, ws).T
    return y if bias is None else y + np.asarray(bias, np.float64)


def mlp(x, w1, s1, w3, s3, w2, s2):
    """SwiGLU MLP of rows x on one expert's 8-bit weights."""
    xv = rows_value(*quantize_rows(x))
    g, u = xv @ weight_value(w1, s1).T, xv @ weight_value(w3, s3).T
    f = g / (1.0 + np.exp(-g)) * u
    return rows_value(*quantize_rows(f)) @ weight_value(w2, s2).T


def route(logits, top_k, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_rule="max", normalize=False,
          scale=1.0):
    """(weights float64, ids) by the definition: experts in order of
    (open, key, lower id)."""
    z = np.asarray(logits, np.float64)
    n, e = z.shape
    b = np.zeros(e) if bias is None else np.asarray(bias, np.float64)
    big = float(np.finfo(np.float32).max)
    avail = ~np.isnan(z) & (z >= -big) & (~np.isnan(b) & (b >= -big))[None, :]
    z = np.where(avail, np.minimum(z, big), 0.0)
    if scoring == "softmax":
        top = np.where(avail, z, -big).max(1, keepdims=True)
        s = np.where(avail, np.exp(np.where(avail, z - top, 0.0)), 0.0)
        s = s / np.maximum(s.sum(1, keepdims=True), 1e-300)
    else:
        with np.errstate(over="ignore"):
            s = np.where(avail, 1.0 / (1.0 + np.exp(-z)), 0.0)
    v = np.where(avail, s + b, -np.inf)
    key = np.where(avail, z, -np.inf) if bias is None else v
    size = e // n_groups
    ids = np.empty((n, top_k), np.int64)
    for r in range(n):
        open_ = np.ones(e, bool)
        if n_groups > 1:
            val = []
            for g in range(n_groups):
                m = slice(g * size, (g + 1) * size)
                if group_rule == "max":
                    val.append(key[r, m].max())
                else:
                    best = np.sort(v[r, m][v[r, m] > -np.inf])[::-1][:2]
                    val.append(best.sum() if best.size else -np.inf)
            kept = sorted(range(n_groups), key=lambda g: (-val[g], g))[:topk_groups]
            open_ = np.isin(np.arange(e) // size, kept)
        order = sorted(np.nonzero(open_)[0], key=lambda i: (-key[r, i], i))
        ids[r] = order[:top_k]
    w = np.take_along_axis(s, ids, 1)
    if normalize:
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-20)
    return w * scale, ids

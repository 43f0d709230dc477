"""A paged key/value cache in 8 bits, attention over it, and the importance of
its tokens (``last_query_importance`` on cached keys).

Values are e4m3 with one power-of-two scale per page and key head, for K and
for V.  Pages hold 32, 64 or 128 tokens; who owns which is the caller's table.
"""

from __future__ import annotations

import ctypes as C

import torch

from .. import _native as N
from .rotary import _strides, overlap, rows_apart, written

TILE = 32
_TAG16 = {torch.float16: N.TM_DT_F16, torch.bfloat16: N.TM_DT_BF16}


def _int32(name: str, t: torch.Tensor, dims: int) -> torch.Tensor:
    if t.dim() != dims or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"Fp8KVCache: {name} must be {dims}-dimensional integers, got {tuple(t.shape)} {t.dtype}")
    # (what 32 bits do not hold stays out of range: as a page that is not there, a length past the table, rows past the call's)
    return t if t.dtype == torch.int32 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


def _scales_hold(scales: torch.Tensor) -> bool:
    """Whether they are powers of two in the range that append writes, or 0 (read on the host)."""
    bits = scales.view(torch.int32)
    return bool((((bits & 0x007fffff) == 0) & (bits >= 27 << 23) & (bits <= 247 << 23) | (bits == 0)).all())


def _rows(t: torch.Tensor):
    """(t [T, H, D] or a copy of it with 16-byte aligned rows, its strides)."""
    if not t.is_contiguous() or t.data_ptr() % 16:
        st, sh = _strides(t)
        if t.stride(2) == 1 and st % 8 == 0 and sh % 8 == 0 and t.data_ptr() % 16 == 0:
            return t, st, sh
        t = t.contiguous()
        t = t if t.data_ptr() % 16 == 0 else t.clone()
    _, h, d = t.shape
    return t, h * d, d


class Fp8KVCache:
    """n_pages pages of page_size tokens for n_kv_heads heads of head_dim key
    columns and v_dim (default head_dim) value columns: (64, 64), (128, 128),
    (192, 128), (192, 192) or (256, 256).

    k and v are [pages, heads, page_size / 32, columns / 32, 64, 16]
    float8_e4m3fn in the order that the matrix instructions read (see
    ``read_pages``), k_scale and v_scale [pages, heads] float32.  They are written
    to in place, not assigned (``wrap`` makes a cache of other storage).

    A batch is given by ``table`` [B, M] (each sequence's pages in order),
    ``lengths`` [B] (its tokens, the new ones counted) and ``starts`` [B + 1]: the
    new tokens of sequence b are rows starts[b] .. starts[b + 1] of the call, its
    last positions; None: one each.  They are int32 on the device (int64 is
    converted) and are read there, so calls need no host synchronisation and can
    be captured.  A page number out of range is a page that is not there.  Calls
    take their scratch from torch's allocator.  Inference only: no gradients."""

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, v_dim: int | None = None, page_size: int = 64,
                 device="cuda"):
        v_dim = head_dim if v_dim is None else v_dim
        self._check(page_size, head_dim, v_dim)
        if n_pages < 1 or n_kv_heads < 1:
            raise ValueError("Fp8KVCache: at least one page and one head")
        shape = lambda d: (n_pages, n_kv_heads, page_size // TILE, d // TILE, 64, 16)  # noqa: E731
        zeros = lambda d: torch.zeros(shape(d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)  # noqa: E731
        ones = lambda: torch.ones((n_pages, n_kv_heads), dtype=torch.float32, device=device)  # noqa: E731
        self._init(zeros(head_dim), zeros(v_dim), ones(), ones())

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "Fp8KVCache":
        """The cache on storage that is there already (k, v, k_scale, v_scale of another one, or kept elsewhere).
        Scales are powers of two from 2^-100 to 2^120, as ``append`` writes them (0 in pages that nobody has written to);
        others are refused.  This reads them once and waits for it; in a stream that is being captured, which cannot
        wait, they are taken as they are."""
        self = cls.__new__(cls)
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 6 or t.dtype != torch.float8_e4m3fn or tuple(t.shape[4:]) != (64, 16) or not t.is_contiguous() \
                    or t.data_ptr() % 16:
                raise ValueError(f"Fp8KVCache: {name} must be [pages, heads, page / 32, columns / 32, 64, 16] "
                                 "float8_e4m3fn, contiguous and 16-byte aligned")
        if k.shape[:3] != v.shape[:3] or k.shape[0] < 1 or k.shape[1] < 1:
            raise ValueError(f"Fp8KVCache: k {tuple(k.shape)} and v {tuple(v.shape)} differ in pages, heads or page size")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.shape != k.shape[:2] or t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError(f"Fp8KVCache: {name} must be {tuple(k.shape[:2])} float32, contiguous")
        self._check(k.shape[2] * TILE, k.shape[3] * TILE, v.shape[3] * TILE)
        self._init(k, v, k_scale, v_scale)
        if not torch.cuda.is_current_stream_capturing() and not _scales_hold(torch.stack((k_scale, v_scale))):
            raise ValueError("Fp8KVCache: scales must be powers of two from 2^-100 to 2^120 (or 0)")
        return self

    @staticmethod
    def _check(page_size, head_dim, v_dim):
        if page_size not in (32, 64, 128):
            raise ValueError(f"Fp8KVCache: page_size {page_size} not in 32, 64, 128")
        if (head_dim, v_dim) not in ((64, 64), (128, 128), (192, 128), (192, 192), (256, 256)):
            raise ValueError(f"Fp8KVCache: columns {(head_dim, v_dim)} not in (64, 64), (128, 128), (192, 128), "
                             "(192, 192), (256, 256)")

    def _init(self, k, v, k_scale, v_scale):
        self.device = N.require_hip(k, v, k_scale, v_scale)
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads = k.shape[:2]
        self.page_size, self.head_dim, self.v_dim = k.shape[2] * TILE, k.shape[3] * TILE, v.shape[3] * TILE
        self._desc = N.Kv8Cache(self.n_pages, self.n_kv_heads, self.head_dim, self.v_dim, self.page_size, k.data_ptr(),
                                v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._ref = C.byref(self._desc)
        self._scale = self.head_dim ** -0.5

    # The calls use these tensors' addresses, so the tensors live as long as the cache and are not exchanged.
    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)

    def read_pages(self, pages: torch.Tensor | None = None):
        """(K [n, heads, page_size, head_dim], V [n, heads, page_size, v_dim]) float32 of the given pages (all)."""
        pick = (lambda t: t) if pages is None else (lambda t: t.view(torch.uint8)[pages].view(t.dtype)  # noqa: E731
                                                    if t.dtype == torch.float8_e4m3fn else t[pages])
        n, h = pick(self.k_scale).shape
        k = pick(self.k).view(n, h, self.page_size // TILE, self.head_dim // TILE, 2, TILE, 16)
        k = k.permute(0, 1, 2, 5, 3, 4, 6).reshape(n, h, self.page_size, self.head_dim)
        v = pick(self.v).view(n, h, self.page_size // TILE, self.v_dim // TILE, 2, TILE, 2, 2, 4)
        v = v.permute(0, 1, 2, 6, 7, 4, 8, 3, 5).reshape(n, h, self.page_size, self.v_dim)
        return k.float() * pick(self.k_scale)[:, :, None, None], v.float() * pick(self.v_scale)[:, :, None, None]

    def _batch(self, table, lengths, starts, n_tokens):
        """(tm_kv8_batch, the tensors that it points to): int32, as they are or converted."""
        dev = self.device
        if table.device != dev or lengths.device != dev or (starts is not None and starts.device != dev):
            N.require_hip(self.k, table, lengths, starts)
        if table.dtype is not torch.int32 or table.dim() != 2:
            table = _int32("table", table, 2)
        if lengths.dtype is not torch.int32 or lengths.dim() != 1:
            lengths = _int32("lengths", lengths, 1)
        b, most = table.shape
        if not table.is_contiguous() and (table.stride(1) != 1 and most > 1 or table.stride(0) < most and b > 1):
            table = table.contiguous()
        if not lengths.is_contiguous():
            lengths = lengths.contiguous()
        if starts is not None:
            starts = _int32("starts", starts, 1).contiguous()
        if lengths.shape[0] != b or (n_tokens != b if starts is None else starts.shape[0] != b + 1):
            raise ValueError(f"Fp8KVCache: table {tuple(table.shape)}, lengths {tuple(lengths.shape)}, starts "
                             f"{None if starts is None else tuple(starts.shape)} and {n_tokens} rows do not go together")
        batch = N.Kv8Batch(table.data_ptr(), table.stride(0) if b > 1 else most, lengths.data_ptr(),
                           None if starts is None else starts.data_ptr(), b, n_tokens, most, 0)
        return batch, (table, lengths, starts)

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               starts: torch.Tensor | None = None) -> None:
        """Writes the new tokens' k [T, heads, head_dim] and v [T, heads, v_dim]
        (float32, float16 or bfloat16) into their pages.  A page's scale is the
        smallest power of two that holds the largest value; where new tokens
        raise it, the page's older values are rounded again; rows of zeros and
        non-finite values alone never do.  A non-finite value is stored as NaN.
        A page that is written belongs to one sequence."""
        n = k.shape[0]
        if k.shape != (n, self.n_kv_heads, self.head_dim) or v.shape != (n, self.n_kv_heads, self.v_dim) \
                or k.dtype is not v.dtype:
            raise ValueError(f"Fp8KVCache.append: k must be [T, {self.n_kv_heads}, {self.head_dim}] and v [T, "
                             f"{self.n_kv_heads}, {self.v_dim}] of one dtype, got {tuple(k.shape)} {k.dtype} and "
                             f"{tuple(v.shape)} {v.dtype}")
        tag = N.dtype_tag(k.dtype)
        dev = self.device
        if k.device != dev or v.device != dev:
            N.require_hip(self.k, k, v)
        batch, kept = self._batch(table, lengths, starts, n)
        k, ks_t, ks_h = _rows(k)
        v, vs_t, vs_h = _rows(v)
        with N.on_device(dev):
            N.call("tm_kv8_append", self._ref, C.byref(batch), tag, k.data_ptr(), ks_t, ks_h, v.data_ptr(), vs_t, vs_h,
                   N.stream(dev))

    def _queries(self, q, scale):
        """(dtype tag, scale) of checked queries."""
        tag = _TAG16.get(q.dtype)
        if tag is None or q.dim() != 3 or q.shape[2] != self.head_dim or q.shape[1] % self.n_kv_heads or q.shape[1] == 0:
            raise ValueError(f"Fp8KVCache: q must be [T, heads, {self.head_dim}] float16 or bfloat16, its heads a "
                             f"multiple of {self.n_kv_heads}, got {tuple(q.shape)} {q.dtype}")
        if q.device != self.device:
            N.require_hip(self.k, q)
        return tag, (self._scale if scale is None else float(scale))

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None, *,
               scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None,
               return_lse: bool = False):
        """softmax(scale q K^T) V [T, heads, v_dim] of the new tokens' q [T,
        heads, head_dim] (float16, bfloat16) over the cached positions of their
        sequences (``append`` first): up to their own with ``causal``, else all.
        scale: positive, default head_dim ** -0.5.  With ``return_lse`` also the
        log sum exp of the scores [T, heads] float32.  A token that sees nothing
        gets zeros and -inf; rows that ``starts`` leaves out are not written.
        ``out`` must not overlap q."""
        tag, scale = self._queries(q, scale)
        n, h, _ = q.shape
        batch, kept = self._batch(table, lengths, starts, n)
        dev = self.device
        q, qs_t, qs_h = _rows(q)
        if out is None:
            out = q.new_empty((n, h, self.v_dim))
            os_t, os_h = h * self.v_dim, self.v_dim
        else:
            N.require_hip(q, out)
            os_t, os_h = _strides(out) if out.dim() == 3 else (0, 0)
            if out.shape != (n, h, self.v_dim) or out.dtype != q.dtype or not rows_apart(out) or out.data_ptr() % 16 \
                    or os_t % 8 or os_h % 8:
                raise ValueError(f"Fp8KVCache.attend: out must be {(n, h, self.v_dim)} {q.dtype} with 16-byte aligned "
                                 "rows that do not overlap")
            if overlap(out, q):
                raise ValueError("Fp8KVCache.attend: out must not overlap q")
            written(out)
        lse = torch.empty((n, h), dtype=torch.float32, device=dev) if return_lse else None
        ref = C.byref(batch)
        nbytes = N.lib().tm_kv8_attention_workspace_size(self._ref, ref, h)
        ws = q.new_empty(nbytes // 2) if nbytes else None
        with N.on_device(dev):
            N.call("tm_kv8_attention", self._ref, ref, tag, q.data_ptr(), qs_t, qs_h, h, scale, 1 if causal else 0,
                   out.data_ptr(), os_t, os_h, N.ptr(lse), N.ptr(ws), nbytes, N.stream(dev))
        return (out, lse) if return_lse else out

    def importance(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                   lse: torch.Tensor | None = None, out_len: int | None = None,
                   starts: torch.Tensor | None = None) -> torch.Tensor:
        """Head mean of the probabilities that one query per sequence, q [B,
        heads, head_dim], gives to each cached position: [B, out_len] float32
        (default: the table's width in tokens), 0 from a sequence's length on.
        With ``starts`` (and out_len, the rows of the call) of the new tokens
        alone: [out_len], row starts[b] + i being position lengths[b] - n + i of
        a sequence with n of them; 0 where a row is no sequence's.
        lse [B, heads] float32: the queries' log sum exp where ``attend`` has
        given it (keys are read once then).  At most 256 heads.
        ``table_moe.utils.importance.cached_importance`` also stores the scores
        for the keep rule."""
        tag, scale = self._queries(q, scale)
        b, h, _ = q.shape
        if starts is not None and out_len is None:
            raise ValueError("Fp8KVCache.importance: starts needs out_len, the number of the call's rows")
        if out_len is not None and int(out_len) < 0:
            raise ValueError("Fp8KVCache.importance: out_len must not be negative")
        batch, kept = self._batch(table, lengths, starts, b if starts is None else int(out_len))
        if batch.n_seqs != b:
            raise ValueError(f"Fp8KVCache.importance: {b} queries for {batch.n_seqs} sequences")
        dev = self.device
        q, qs_t, qs_h = _rows(q)
        out_len = batch.max_pages * self.page_size if out_len is None else int(out_len)
        out = torch.empty((b, out_len), dtype=torch.float32, device=dev) if starts is None else \
            torch.zeros(out_len, dtype=torch.float32, device=dev)
        ref, ld_lse, ws, nbytes = C.byref(batch), 0, None, 0
        if lse is not None:
            N.require_hip(q, lse)
            if lse.shape != (b, h) or lse.dtype != torch.float32:
                raise ValueError(f"Fp8KVCache.importance: lse must be {(b, h)} float32")
            if lse.stride(1) != 1 and h > 1 or lse.stride(0) < h and b > 1:
                lse = lse.contiguous()
            ld_lse = lse.stride(0) if b > 1 else h
        else:
            nbytes = N.lib().tm_kv8_importance_workspace_size(self._ref, ref, h)
            ws = q.new_empty(nbytes // 2) if nbytes else None
        with N.on_device(dev):
            if starts is None:
                N.call("tm_kv8_importance", self._ref, ref, tag, q.data_ptr(), qs_t, qs_h, h, scale, N.ptr(lse), ld_lse,
                       out_len, out.data_ptr(), out_len, N.ptr(ws), nbytes, N.stream(dev))
            else:
                N.call("tm_kv8_importance_rows", self._ref, ref, tag, q.data_ptr(), qs_t, qs_h, h, scale, N.ptr(lse),
                       ld_lse, out.data_ptr(), N.ptr(ws), nbytes, N.stream(dev))
        return out

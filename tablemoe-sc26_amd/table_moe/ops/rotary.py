"""Rotary positions with several axes: text, images (row, column) and video
(time, row, column), for the queries and keys whose scores the importance and
the attention of this package take.

One tm_rotate_positions call turns q and k: angles in 64 bits, the rotation in
fp32, one rounding.  It is differentiable (the gradient is the rotation back, a
tangent is turned as its tensor is).
"""

from __future__ import annotations

import ctypes as C
import functools
import math

import torch
from torch.autograd.forward_ad import unpack_dual

from .. import _native as N

_INTEGERS = (torch.int64, torch.int32)


@functools.lru_cache(maxsize=64)
def _sections(sections: tuple):
    return (C.c_int32 * len(sections))(*sections)


def rows_apart(t: torch.Tensor) -> bool:
    """Whether the [T, H, D] view's rows of D do not overlap each other."""
    (n, h, d), (st, sh, sd) = t.shape, t.stride()
    if sd != 1 and d > 1:
        return False
    pairs = sorted((s, m) for s, m in ((st, n), (sh, h)) if m > 1)
    end = d
    for s, m in pairs:
        if s < end:
            return False
        end = s * (m - 1) + end
    return True


def _span(t: torch.Tensor):
    last = sum((m - 1) * s for m, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def written(*tensors) -> None:
    """Tells autograd, for a graph that has saved one of them (an error in its backward, as after any write in place)."""
    for t in tensors:
        if t is None or t.is_inference():
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("out has no gradient")
        torch.autograd.graph.increment_version(t)


def overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether the [T, H, D] views may share memory; views of one fused projection's rows that take different columns do
    not, be they next to each other ([T, H + Hkv, D]) or by turns ([T, H, 2, D]); nor do heads of a buffer by heads."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    (a, b), (c, d) = _span(x), _span(y)
    if a >= d or c >= b:
        return False
    steps = [[t.stride(i) * t.element_size() for t in (x, y) if t.shape[i] > 1] for i in (0, 1)]
    step = math.gcd(*steps[0], *steps[1])  # each view's rows start at one place modulo this
    if step and x.shape[2] * x.element_size() <= (c - a) % step <= step - y.shape[2] * y.element_size():
        return False
    for i in (0, 1):  # what a token (or head) takes, modulo the distance between them
        if len(set(steps[i])) == 1 and steps[i][0]:
            step, (a, b), (c, d) = steps[i][0], _span(x.select(i, 0)), _span(y.select(i, 0))
            if b - a <= (c - a) % step <= step - (d - c):
                return False
    return True


def _itself(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether views of one shape are the same elements (the stride of a single token or head means nothing)."""
    return x.data_ptr() == y.data_ptr() and all(m == 1 or s == t for m, s, t in zip(x.shape, x.stride(), y.stride()))


def _check_out(name: str, out: torch.Tensor, x: torch.Tensor, others) -> None:
    if not (out is x and x.is_contiguous()):
        if out.shape != x.shape or out.dtype != x.dtype or not rows_apart(out):
            raise ValueError(f"rotate_positions: {name} must be {tuple(x.shape)} {x.dtype} with unit stride along its last "
                             "dimension and rows that do not overlap")
        if not _itself(out, x) and overlap(out, x):
            raise ValueError(f"rotate_positions: {name} may be the input itself, not overlap it otherwise")
    if any(overlap(out, t) for t in others):
        raise ValueError(f"rotate_positions: {name} overlaps the other input or output")


def _strides(t: torch.Tensor):
    st, sh, _ = t.stride()
    return st if t.shape[0] > 1 else 0, sh if t.shape[1] > 1 else 0


def _run(q, k, positions, inv_freq, sections, interleaved, adjacent, inverse, q_out, k_out, dev):
    n, h, d = q.shape
    qs_t, qs_h, _ = q.stride()
    qo_t, qo_h, _ = q_out.stride()
    kp = kv = ks_t = ks_h = kop = ko_t = ko_h = 0
    if k is not None:
        kp, kv, kop = k.data_ptr(), k.shape[1], k_out.data_ptr()
        ks_t, ks_h, _ = k.stride()
        ko_t, ko_h, _ = k_out.stride()
    axes = len(sections)
    with N.on_device(dev):
        N.call("tm_rotate_positions", N.dtype_tag(q.dtype), q.data_ptr(), n, h, qs_t, qs_h, kp, kv, ks_t, ks_h, d,
               2 * inv_freq.shape[0], positions.data_ptr(), positions.stride(0) if axes > 1 else n, axes,
               _sections(sections), interleaved, adjacent, inverse, inv_freq.data_ptr(), q_out.data_ptr(), qo_t, qo_h,
               kop, ko_t, ko_h, N.stream(dev))


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() or t.stride(2) == 1 else t.contiguous()


def _new(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, how):
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)
        ctx.how = how
        qq = _unit_rows(q)
        kk = None if k is None else _unit_rows(k)
        q_out, k_out = _new(qq), None if k is None else _new(kk)
        _run(qq, kk, positions, inv_freq, *how, q_out, k_out, q.device)
        return q_out, k_out

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        positions, inv_freq = ctx.saved_tensors
        return _Rotate.apply(tq, tk, positions, inv_freq, ctx.how)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        sections, interleaved, adjacent, inverse = ctx.how
        how = (sections, interleaved, adjacent, 1 - inverse)
        # (the gradient of the part that is not asked for is not computed)
        if not ctx.needs_input_grad[0]:
            return None, _Rotate.apply(dk, None, positions, inv_freq, how)[0], None, None, None
        dq, dk = _Rotate.apply(dq, dk if ctx.needs_input_grad[1] else None, positions, inv_freq, how)
        return dq, dk, None, None, None


def _dual(t) -> bool:
    """Whether it carries a tangent (which requires_grad does not say)."""
    return t is not None and unpack_dual(t).tangent is not None


def rotate_positions(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
                     sections=None, *, interleaved: bool = False, adjacent: bool = False, inverse: bool = False,
                     out=None):
    """(q', k') of q [T, H, D] and k [T, Hkv, D] (or None), float32, float16 or
    bfloat16, any strides with unit stride along D (others are copied).

    positions: [A, T] integers, or [T] for one axis.  inv_freq [R / 2] float32:
    frequency i turns with axis a(i); columns R .. D are copied.  sections (A
    numbers summing to R / 2; default: all of one axis): runs of frequencies in
    the axes' order; with ``interleaved`` a(i) = i % A where i < A * sections[i %
    A], else 0.  Pairs are columns (i, i + R / 2), or (2i, 2i + 1) with
    ``adjacent``.  ``inverse`` turns back.  angle = positions * inv_freq in 64
    bits, the rest in fp32, rounded once.

    out: a pair (q_out, k_out) to write to, which may be (q, k) themselves; then
    there are no gradients.  Otherwise gradients of any order flow to q and k, in
    reverse and (torch.autograd.forward_ad) forward mode."""
    dev = N.require_hip(q, k, positions, inv_freq)
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]
                                           or k.dtype is not q.dtype)):
        raise ValueError("rotate_positions expects q [T, H, D] and k [T, Hkv, D] of one dtype")
    n = q.shape[0]
    if positions.dim() == 1:
        positions = positions[None]
    axes = positions.shape[0]
    if positions.dim() != 2 or positions.shape[1] != n or positions.dtype not in _INTEGERS:
        raise ValueError(f"rotate_positions: positions must be [A, {n}] or [{n}] integers, got {tuple(positions.shape)} "
                         f"{positions.dtype}")
    if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float32 or inv_freq.requires_grad and torch.is_grad_enabled() \
            or _dual(inv_freq):
        raise ValueError("rotate_positions: inv_freq must be [R / 2] float32 and has no gradient")
    sections = (inv_freq.shape[0],) if sections is None else tuple(map(int, sections))
    if len(sections) != axes:
        raise ValueError(f"rotate_positions: {len(sections)} sections for {axes} axes")
    if positions.dtype is not torch.int64:
        positions = positions.long()
    if not positions.is_contiguous() and (positions.stride(1) != 1 and n > 1 or positions.stride(0) < n and axes > 1):
        positions = positions.contiguous()
    if not inv_freq.is_contiguous():
        inv_freq = inv_freq.contiguous()
    how = (sections, 1 if interleaved else 0, 1 if adjacent else 0, 1 if inverse else 0)
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled() or _dual(q) or _dual(k):
        if out is not None:
            raise ValueError("rotate_positions: no gradients through out")
        return _Rotate.apply(q, k, positions, inv_freq, how)
    q, k = _unit_rows(q), None if k is None else _unit_rows(k)
    if out is None:
        q_out, k_out = _new(q), None if k is None else _new(k)
    else:
        q_out, k_out = out
        if (k is None) != (k_out is None):
            raise ValueError("rotate_positions: out holds a tensor for each of q and k")
        N.require_hip(q, q_out, k_out)
        if _dual(q_out) or _dual(k_out):
            raise ValueError("out has no gradient")
        _check_out("out[0]", q_out, q, () if k is None else (k, k_out))
        if k is not None:
            _check_out("out[1]", k_out, k, (q,))
        written(q_out, k_out)
    _run(q, k, positions, inv_freq, *how, q_out, k_out, dev)
    return q_out, k_out

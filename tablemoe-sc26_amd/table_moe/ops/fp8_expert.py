"""SwiGLU experts on 8-bit weights: the 8-bit forms of ``GroupedExperts`` and
``SharedExperts`` (same calls; GlobalTable.layer_forward_recompute takes
either).

Weights are e4m3 as nn.Linear stores them, w1, w3 [E, I, H] and w2 [E, H, I],
each with one fp32 scale per block of 128 x 128.  Activations are quantised in
the call in blocks of 128 columns (the rule of ``quantize_rows_fp8``), and so
is f = silu(x W1^T) * (x W3^T), which stays fp32 until then; y is rounded once.
"""

from __future__ import annotations

import ctypes as C

import torch

from .. import _native as N
from .fp8_blocks import BLOCK, aligned, check_weight, quantize_weight_fp8


def _descriptor(name, w1, s1, w3, s3, w2, s2):
    """(kept tensors, tm_fp8_experts) of checked weights [E, I, H] / [E, H, I]."""
    N.require_hip(w1, s1, w3, s3, w2, s2)
    if w1.dim() != 3:
        raise ValueError(f"{name}: w1 must be [E, I, H], got {tuple(w1.shape)}")
    e, inter, h = w1.shape
    if h % BLOCK or inter % BLOCK:
        raise ValueError(f"{name}: hidden and intermediate sizes must be multiples of {BLOCK}")
    check_weight(name, w1, s1, (e, inter, h))
    check_weight(name, w3, s3, (e, inter, h))
    check_weight(name, w2, s2, (e, h, inter))
    kept = [aligned(w1), s1.contiguous(), aligned(w3), s3.contiguous(), aligned(w2), s2.contiguous()]
    return kept, N.Fp8Experts(e, h, inter, 0, *(t.data_ptr() for t in kept))


def _row_stride(t: torch.Tensor, width: int) -> int:
    """t's row stride; a single row's own means nothing (it may be odd, or 0)."""
    return t.stride(0) if t.shape[0] > 1 else width


def _rows(x: torch.Tensor, width: int):
    """(x or an aligned copy, its row stride) for rows of ``width`` elements."""
    ld = _row_stride(x, width)
    if x.stride(1) != 1 or ld % 8 or ld < width or x.data_ptr() % 16:
        x = aligned(x)
        ld = _row_stride(x, width)
    return x, ld


class Fp8GroupedExperts:
    """Stacked 8-bit expert weights; one tm_fp8_grouped_swiglu call per forward
    (grouping included).  Scratch comes from torch's allocator in each call, so
    calls on several streams and captured graphs do not share any."""

    def __init__(self, w1, s1, w3, s3, w2, s2):
        self._kept, self._desc = _descriptor("Fp8GroupedExperts", w1, s1, w3, s3, w2, s2)
        self._ref = C.byref(self._desc)
        self.n_experts, self.inter, self.hidden = w1.shape
        self.device = w1.device
        self._sizes: dict = {}

    @classmethod
    def from_weights(cls, w1, w3, w2) -> "Fp8GroupedExperts":
        """The experts of float weights, quantised here."""
        return cls(*quantize_weight_fp8(w1), *quantize_weight_fp8(w3), *quantize_weight_fp8(w2))

    def _workspace(self, n, k):
        nbytes = self._sizes.get((n, k))
        if nbytes is None:
            if len(self._sizes) >= 256:
                self._sizes.clear()
            nbytes = self._sizes[(n, k)] = max(N.lib().tm_fp8_grouped_swiglu_workspace_size(self._ref, n, k), 1)
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device)

    def forward(self, hidden: torch.Tensor, ids: torch.Tensor, mask: torch.Tensor, slot_out: torch.Tensor):
        """slot_out[b, s] = expert(ids[b, s]) MLP of hidden[b] for masked pairs
        (others untouched); ``mask`` is [N, k] or a per-token [N] flag; returns
        slot_out."""
        N.require_hip(hidden, ids, mask, slot_out, self._kept[0])
        dt = hidden.dtype
        if dt not in (torch.float16, torch.bfloat16) or slot_out.dtype != dt:
            raise ValueError("hidden and slot_out must share dtype float16 or bfloat16")
        n, k = ids.shape
        if hidden.shape != (n, self.hidden):
            raise ValueError(f"hidden must be [{n}, {self.hidden}], got {tuple(hidden.shape)}")
        if mask.shape != (n,) and mask.shape != (n, k):
            raise ValueError(f"mask must be [{n}] or [{n}, {k}], got {tuple(mask.shape)}")
        if slot_out.shape != (n, k, self.hidden) or slot_out.stride(-1) != 1:
            raise ValueError(f"slot_out must be [N, {k}, {self.hidden}] with unit stride along hidden")
        so_b, so_s = slot_out.stride(0) if n > 1 else 0, slot_out.stride(1) if k > 1 else 0
        if so_b % 8 or so_s % 8 or slot_out.data_ptr() % 16:
            raise ValueError("slot_out rows must start on 16-byte boundaries (strides multiples of 8 elements)")
        if (n > 1 and so_b < self.hidden) or (k > 1 and so_s < self.hidden) or (n > 1 and k > 1 and so_b == so_s):
            raise ValueError("slot_out rows must not overlap")
        if ids.dtype != torch.long or ids.stride(1) != 1 or ids.stride(0) < k:  # (stride 0: one row for all tokens)
            ids = ids.long().contiguous()
        x, ld = _rows(hidden, self.hidden)
        m = N.as_u8(mask)
        ms_b, ms_s = (m.stride(0), 0) if m.dim() == 1 else (m.stride(0), m.stride(1))
        with N.on_device(self.device):
            ws = self._workspace(n, k)
            N.call("tm_fp8_grouped_swiglu", self._ref, N.dtype_tag(dt), x.data_ptr(), n, ld, ids.data_ptr(), k,
                   max(ids.stride(0), k), m.data_ptr(), ms_b, ms_s, slot_out.data_ptr(), so_b, so_s, ws.data_ptr(),
                   ws.numel(), N.stream(self.device))
        return slot_out


class Fp8SharedExperts:
    """One dense SwiGLU MLP on 8-bit weights w1, w3 [I, H] and w2 [H, I] run
    over every row (a layer's shared experts); one tm_fp8_expert_swiglu call."""

    def __init__(self, w1, s1, w3, s3, w2, s2):
        if w1.dim() != 2:
            raise ValueError(f"Fp8SharedExperts: w1 must be [I, H], got {tuple(w1.shape)}")
        self._kept, self._desc = _descriptor("Fp8SharedExperts", *(t.unsqueeze(0) for t in (w1, s1, w3, s3, w2, s2)))
        self._ref = C.byref(self._desc)
        self.inter, self.hidden = w1.shape
        self.device = w1.device

    @classmethod
    def from_weights(cls, w1, w3, w2) -> "Fp8SharedExperts":
        return cls(*quantize_weight_fp8(w1), *quantize_weight_fp8(w3), *quantize_weight_fp8(w2))

    def forward(self, hidden: torch.Tensor, out: torch.Tensor | None = None,
                addend: torch.Tensor | None = None) -> torch.Tensor:
        """y = MLP(hidden) [M, H], or dtype(addend + MLP) with ``addend`` [M, H]
        (not overlapping ``out``) in one rounding."""
        N.require_hip(hidden, out, addend, self._kept[0])
        dt = hidden.dtype
        if dt not in (torch.float16, torch.bfloat16) or hidden.dim() != 2 or hidden.shape[1] != self.hidden:
            raise ValueError(f"hidden must be [M, {self.hidden}] float16 or bfloat16")
        m, h = hidden.shape
        if out is None:
            out = torch.empty((m, h), dtype=dt, device=self.device)
        for name, t in (("out", out), ("addend", addend)):
            if t is not None and (t.shape != (m, h) or t.dtype != dt or t.stride(1) != 1 or _row_stride(t, h) % 8
                                  or _row_stride(t, h) < h or t.data_ptr() % 16):
                raise ValueError(f"{name} must be [{m}, {h}] {dt} with 16-byte aligned rows")
        x, ld = _rows(hidden, h)
        with N.on_device(self.device):
            nbytes = N.lib().tm_fp8_expert_swiglu_workspace_size(self._ref, m)
            ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=self.device)
            N.call("tm_fp8_expert_swiglu", self._ref, N.dtype_tag(dt), x.data_ptr(), m, ld, N.ptr(addend),
                   0 if addend is None else _row_stride(addend, h), out.data_ptr(), _row_stride(out, h),
                   ws.data_ptr(), ws.numel(), N.stream(self.device))
        return out

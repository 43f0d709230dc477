"""8-bit values (e4m3) with a scale per block of 128: quantisers and a linear layer.

Activations carry one fp32 scale per row and 128 columns, weights one per
block of 128 x 128; a value stands for q * scale.  The quantisers choose powers
of two, so dividing by the scale is exact; the products take any fp32 scales,
such as those a checkpoint brings.
"""

from __future__ import annotations

import torch

from .. import _native as N

BLOCK = 128


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def quantize_rows_fp8(x: torch.Tensor):
    """x [M, K] (float32, float16 or bfloat16) -> (q [M, K] float8_e4m3fn,
    scale [M, ceil(K/128)] float32).  Rows of q are stored padded with zeros to
    whole blocks: for K no multiple of 128, q is a view of a wider tensor."""
    if x.dim() != 2:
        raise ValueError(f"quantize_rows_fp8 expects a 2D tensor, got {tuple(x.shape)}")
    dev = N.require_hip(x)
    tag = N.dtype_tag(x.dtype)
    m, k = x.shape
    if k == 0:
        raise ValueError("quantize_rows_fp8: no columns")
    if x.stride(1) != 1 or x.stride(0) < k:
        x = x.contiguous()
    kb = blocks(k)
    q = torch.empty((m, kb * BLOCK), dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty((m, kb), dtype=torch.float32, device=dev)
    with N.on_device(dev):
        N.call("tm_fp8_quantize_rows", tag, N.ptr(x), m, k, max(x.stride(0), k), N.ptr(q), kb * BLOCK, N.ptr(scale), kb,
               N.stream(dev))
    return (q if k == kb * BLOCK else q[:, :k]), scale


def quantize_weight_fp8(w: torch.Tensor):
    """w [N, K] or [E, N, K] -> (q of its shape float8_e4m3fn, scale [(E,)
    ceil(N/128), ceil(K/128)] float32).  For K no multiple of 128, q is a view
    of a wider tensor, whose rows are padded with zeros."""
    if w.dim() not in (2, 3):
        raise ValueError(f"quantize_weight_fp8 expects [N, K] or [E, N, K], got {tuple(w.shape)}")
    dev = N.require_hip(w)
    tag = N.dtype_tag(w.dtype)
    n, k = w.shape[-2:]
    if n == 0 or k == 0:
        raise ValueError("quantize_weight_fp8: an empty matrix")
    mats = w.shape[0] if w.dim() == 3 else 1
    w = w.contiguous()
    nb, kb = blocks(n), blocks(k)
    lead = (mats,) if w.dim() == 3 else ()
    q = torch.empty((*lead, n, kb * BLOCK), dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty((*lead, nb, kb), dtype=torch.float32, device=dev)
    with N.on_device(dev):
        N.call("tm_fp8_quantize_weight", tag, N.ptr(w), mats, n, k, N.ptr(q), kb * BLOCK, N.ptr(scale), N.stream(dev))
    return (q if k == kb * BLOCK else q[..., :k]), scale


def check_weight(name: str, q: torch.Tensor, scale: torch.Tensor, shape: tuple) -> None:
    """An 8-bit weight of ``shape`` [..., N, K] and its block scales."""
    if q.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        raise ValueError(f"{name}: weights must be float8_e4m3fn with float32 scales, got {q.dtype} and {scale.dtype}")
    want = (*shape[:-2], blocks(shape[-2]), blocks(shape[-1]))
    if tuple(q.shape) != tuple(shape) or tuple(scale.shape) != want:
        raise ValueError(f"{name}: expected weight {tuple(shape)} with scales {want}, got {tuple(q.shape)} and "
                         f"{tuple(scale.shape)}")


def aligned(q: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned (itself, or a copy)."""
    q = q.contiguous()
    return q if q.data_ptr() % 16 == 0 else q.clone()


class Fp8Linear:
    """y = x W^T + bias on an 8-bit weight [N, K] with block scales
    [ceil(N/128), ceil(K/128)].

    ``forward`` quantises x [..., K] (float32, float16, bfloat16) in the call, or
    takes the pair that ``quantize_rows_fp8`` returns, with ``dtype`` naming the
    output's; sums are fp32, y is rounded once (a bias of another type than the
    output's is rounded to it first).  float32 outputs take every
    product exactly; 16-bit ones may run on the 8-bit matrix instructions (an
    error of up to 6e-5 of a sum's size before the rounding).  A weight whose
    K is no multiple of 128 is copied once to padded rows.  Calls allocate
    their scratch from torch's allocator: they can be captured in graphs and
    made on any stream.  ``out`` must not overlap x."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None):
        if weight.dim() != 2:
            raise ValueError(f"Fp8Linear: weight must be [N, K], got {tuple(weight.shape)}")
        self.device = N.require_hip(weight, scale, bias)
        self.out_features, self.in_features = weight.shape
        check_weight("Fp8Linear", weight, scale, tuple(weight.shape))
        if bias is not None and bias.shape != (self.out_features,):
            raise ValueError(f"Fp8Linear: bias must be [{self.out_features}], got {tuple(bias.shape)}")
        kp = blocks(self.in_features) * BLOCK
        if kp == self.in_features:
            self.weight = aligned(weight)
        else:
            self.weight = torch.zeros((self.out_features, kp), dtype=torch.uint8, device=self.device)
            self.weight[:, :self.in_features] = weight.view(torch.uint8)
        self.scale, self.bias = scale.contiguous(), bias

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "Fp8Linear":
        """The layer of a float weight [N, K], quantised here."""
        return cls(*quantize_weight_fp8(weight), bias)

    def _bias_of(self, dtype):
        return None if self.bias is None else self.bias.to(dtype).contiguous()

    def forward(self, x, out: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
        k, n = self.in_features, self.out_features
        xs = None
        if isinstance(x, (tuple, list)):
            x, xs = x
            if dtype is None and out is None:
                raise ValueError("Fp8Linear: name the output's dtype for quantised x")
            dtype = out.dtype if dtype is None else dtype
            N.require_hip(x, xs, self.weight)
            if x.dtype != torch.float8_e4m3fn or xs.dtype != torch.float32 or x.dim() != 2 or xs.shape != (x.shape[0],
                                                                                                      blocks(k)):
                raise ValueError("Fp8Linear: quantised x is the pair that quantize_rows_fp8 returns")
            kp = blocks(k) * BLOCK
            if x.stride(1) != 1 or x.stride(0) < kp or x.stride(0) % 16 or x.data_ptr() % 16 or xs.stride(1) != 1:
                raise ValueError("Fp8Linear: rows of quantised x must be padded to whole blocks, 16-byte aligned, as "
                                 "quantize_rows_fp8 returns them")
            end = x.storage_offset() + (x.shape[0] - 1) * x.stride(0) + kp  # (one byte an element)
            if x.shape[0] > 0 and end > x.untyped_storage().nbytes():
                raise ValueError("Fp8Linear: the last row of quantised x ends before its last block does")
        else:
            N.require_hip(x, self.weight)
            if dtype is not None and dtype != x.dtype:
                raise ValueError("Fp8Linear: the output has x's dtype")
            dtype = x.dtype
        tag = N.dtype_tag(dtype)
        if x.shape[-1] != k:
            raise ValueError(f"Fp8Linear: x must have {k} columns, got {tuple(x.shape)}")
        lead = x.shape[:-1]
        x2 = x if x.dim() == 2 else x.reshape(-1, k)
        if x2.stride(1) != 1 or (x2.stride(0) < k and x2.shape[0] > 1):
            x2 = x2.contiguous()
        m = x2.shape[0]
        if out is None:
            out = torch.empty((*lead, n), dtype=dtype, device=self.device)
        else:
            N.require_hip(out, x2)
            if out.shape != (*lead, n) or out.dtype != dtype:
                raise ValueError(f"Fp8Linear: out must be {(*lead, n)} {dtype}")
        if out.dim() != 2 and not out.is_contiguous():
            raise ValueError("Fp8Linear: out of more or less than two dimensions must be contiguous")
        o2 = out if out.dim() == 2 else out.view(-1, n)
        if m > 0 and (o2.stride(1) != 1 and n > 1 or m > 1 and o2.stride(0) < n):
            raise ValueError("Fp8Linear: out needs a unit stride along its columns and rows that do not overlap")
        ld_x = max(x2.stride(0), k) if xs is None else x2.stride(0)
        with N.on_device(self.device):
            nbytes = N.lib().tm_fp8_linear_workspace_size(m, k, tag)
            ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=self.device)
            bias = self._bias_of(dtype)
            N.call("tm_fp8_linear", tag, N.ptr(x2), N.ptr(xs), m, k, ld_x, 0 if xs is None else xs.stride(0),
                   N.ptr(self.weight), N.ptr(self.scale), n, N.ptr(bias), N.ptr(o2),
                   max(o2.stride(0), n), N.ptr(ws), ws.numel(), N.stream(self.device))
        return out

    __call__ = forward

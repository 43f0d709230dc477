"""The 8-bit quantisers, linear layer and expert MLPs against their definitions
in 64 bits (fp8_ref).

Tolerances.  The quantisers divide by powers of two and round once: equal.  A
sum of K exact products in fp32, block sums scaled and added, is within
(K + 3 K / 128) 2^-24 of the sum of its terms' sizes (one rounding per addition
and per scaling).  The 8-bit matrix instructions, which 16-bit outputs may use,
add the products of 8 consecutive columns aligned to the largest: with 2^E its
exponent (the sum of its factors' exponents, so the product is 2^E or more)
they drop what lies under 2^(E - 13) of each.  The largest is a multiple of
2^(E - 6) and loses nothing, each of the 7 others less than 2^-13 of it: 7 *
2^-13 times the sum over the groups of 8 of their largest product.  An output is
rounded once: half a step, eps / 2.  In the MLP, a value of f that lies within its own error of a
border between two 8-bit values may come out as either: those, and only those,
may add a step times their weight."""

import numpy as np
import pytest
import torch

import fp8_ref as R
from table_moe.ops import (Fp8GroupedExperts, Fp8Linear, Fp8SharedExperts, quantize_rows_fp8, quantize_weight_fp8)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _truncated(x, w):
    """What the 8-bit instructions may drop of x w^T: see above."""
    x, w = np.abs(x), np.abs(w)
    k = x.shape[1]
    out = np.zeros((x.shape[0], w.shape[0]))
    top = np.empty_like(out)
    for k0 in range(0, k, 8):
        top[:] = 0
        for i in range(k0, min(k0 + 8, k)):
            np.maximum(top, np.multiply.outer(x[:, i], w[:, i]), out=top)
        out += top
    return 7 * 2.0 ** -13 * out


def _np(t):
    return t.detach().cpu().double().numpy()


def _rand(seed, *shape, dtype=torch.float32, dev="cuda", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(shape[-1], generator=g)) * scale
    return x.to(dtype).to(dev)


def _w8(seed, *shape, dev="cuda"):
    """8-bit weights with scales that are no powers of two."""
    g = torch.Generator().manual_seed(seed)
    *lead, n, k = shape
    q = (90 * torch.randn(*shape, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = 0.02 / 90 * torch.exp(0.3 * torch.randn(*lead, -(-n // 128), -(-k // 128), generator=g))
    return q.to(dev), s.to(dev)


# ---------------------------------------------------------------- quantisers
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 128), (17, 130), (5, 1000), (64, 2048), (33, 257)])
def test_quantize_rows(hip_device, dtype, m, k):
    x = _rand(m * 31 + k, m, k, dtype=dtype) * 3
    if m > 2:
        x[1] = 0
        x[2, : k // 2] = 0
    q, s = quantize_rows_fp8(x)
    want_q, want_s = R.quantize_rows(_np(x))
    assert q.shape == (m, k) and s.shape == (m, -(-k // 128)) and q.dtype == torch.float8_e4m3fn
    np.testing.assert_array_equal(_np(s), want_s)
    np.testing.assert_array_equal(_np(q.float()), want_q)


def test_quantize_rows_every_border(hip_device):
    """Every midpoint between two 8-bit values and its neighbours, at several scales."""
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (v[1:] + v[:-1]) / 2
    pts = torch.cat([v, mid, torch.nextafter(mid, torch.tensor(1e9)), torch.nextafter(mid, torch.tensor(-1e9))])
    pts = torch.cat([pts, -pts])
    pts = torch.nn.functional.pad(pts, (0, -len(pts) % 64)).view(-1, 64)
    x = torch.cat([pts, torch.full((pts.shape[0], 64), 448.0)], 1)  # the block's largest: scale 1
    for p in (0, -20, 30, -100):
        y = (x.double() * 2.0 ** p).float().to(hip_device)
        q, s = quantize_rows_fp8(y)
        want_q, want_s = R.quantize_rows(_np(y))
        np.testing.assert_array_equal(_np(s), want_s)
        np.testing.assert_array_equal(_np(q.float()), want_q)


def test_quantize_rows_extremes(hip_device):
    x = torch.zeros(8, 256)
    x[0, 0], x[1, 0] = 3.4028234663852886e38, -448.0001
    x[2, 0], x[3, 0] = 1e-45, 1.2e-38
    x[4, :3] = torch.tensor([float("inf"), 1.0, -2.0])
    x[5, :3] = torch.tensor([float("nan"), 1.0, float("-inf")])
    x[6, :128] = float("nan")
    x[7, 127], x[7, 128] = 448.0, 449.0
    q, s = quantize_rows_fp8(x.to(hip_device))
    want_q, want_s = R.quantize_rows(x.double().numpy())
    np.testing.assert_array_equal(_np(s), want_s)
    np.testing.assert_array_equal(_np(q.float()), want_q)


def test_quantize_rows_strides_and_empty(hip_device):
    x = _rand(1, 9, 300)
    wide = torch.full((9, 333), 7.0, device=hip_device)
    wide[:, 5:305] = x
    for v in (wide[:, 5:305], x.t().contiguous().t()):
        q, s = quantize_rows_fp8(v)
        q0, s0 = quantize_rows_fp8(x)
        assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)
    q, s = quantize_rows_fp8(x[:0])
    assert q.shape == (0, 300) and s.shape == (0, 3)
    # the padding of a row is zeros
    q, _ = quantize_rows_fp8(x)
    full = torch.as_strided(q.view(torch.uint8), (9, 384), (384, 1))
    assert int(full[:, 300:].max()) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(128, 128), (3, 130, 257), (1, 1, 1), (2, 300, 384), (5, 64)])
def test_quantize_weight(hip_device, dtype, shape):
    w = _rand(sum(shape), *shape, dtype=dtype, scale=0.02)
    q, s = quantize_weight_fp8(w)
    w3, q3 = w.reshape(-1, *shape[-2:]), q.reshape(-1, *shape[-2:])
    s3 = s.reshape(-1, *s.shape[-2:])
    assert q.shape == shape
    for i in range(w3.shape[0]):
        want_q, want_s = R.quantize_weight(_np(w3[i]))
        np.testing.assert_array_equal(_np(s3[i]), want_s)
        np.testing.assert_array_equal(_np(q3[i].float()), want_q)


# -------------------------------------------------------------------- linear
def _linear_tol(x, wq, ws, y, dtype):
    xv, wv = np.abs(R.rows_value(*R.quantize_rows(x))), np.abs(R.weight_value(wq, ws))
    size = xv @ wv.T
    k = x.shape[1]
    tol = (k + 3 * -(-k // 128)) * U * size + 1e-37
    if dtype != torch.float32:
        tol = tol + _truncated(xv, wv)
    return tol + torch.finfo(dtype).eps / 2 * (np.abs(y) + tol)


def _check_linear(x, wq, ws, bias=None, out=None):
    layer = Fp8Linear(wq, ws, bias)
    got = layer.forward(x, out)
    want = R.linear(_np(x), _np(wq.float()), _np(ws), None if bias is None else _np(bias))
    tol = _linear_tol(_np(x), _np(wq.float()), _np(ws), want, x.dtype)
    if x.dtype == torch.float16:  # values under fp16's smallest normal: half of its smallest step
        tol = tol + 2.0 ** -25
    assert got.dtype == x.dtype
    bad = np.abs(_np(got) - want) > tol
    assert not bad.any(), (np.abs(_np(got) - want)[bad].max(), tol[bad].min(), int(bad.sum()))
    return layer, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n,bias", [
    (1, 128, 16, False), (1, 2048, 1000, True), (3, 256, 1, True), (16, 384, 130, False), (17, 1000, 257, True),
    (33, 64, 48, False), (64, 640, 256, True), (100, 2560, 128, False), (129, 512, 300, True), (257, 256, 512, True),
    (300, 1152, 384, False), (520, 128, 129, False),
])
def test_linear(hip_device, dtype, m, k, n, bias):
    x = _rand(m + k, m, k, dtype=dtype)
    wq, ws = _w8(n, n, k)
    _check_linear(x, wq, ws, _rand(n + 1, n, dtype=dtype) if bias else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_large(hip_device, dtype):
    """Whole tiles and their edges, many of them."""
    x = _rand(2, 1100, 768, dtype=dtype)
    wq, ws = _w8(3, 1300, 768)
    _check_linear(x, wq, ws, _rand(4, 1300, dtype=dtype))


def test_linear_strides_dims_and_out(hip_device):
    x = _rand(5, 40, 512, dtype=torch.bfloat16)
    wq, ws = _w8(6, 200, 512)
    layer, y0 = _check_linear(x, wq, ws)
    wide = torch.zeros(40, 700, dtype=torch.bfloat16, device=hip_device)
    wide[:, 3:515] = x
    assert torch.equal(layer.forward(wide[:, 3:515]), y0)          # rows not 16-byte aligned
    assert torch.equal(layer.forward(x.t().contiguous().t()), y0)  # columns first
    assert torch.equal(layer.forward(x.view(5, 8, 512)), y0.view(5, 8, 200))
    big = torch.full((42, 333), 7.0, dtype=torch.bfloat16, device=hip_device)
    layer.forward(x, out=big[1:41, 100:300])
    assert torch.equal(big[1:41, 100:300], y0)
    rest = big.clone()
    rest[1:41, 100:300] = 7.0
    assert bool((rest == 7.0).all())                               # nothing past the rows and columns
    assert layer.forward(x[:0]).shape == (0, 200)
    assert torch.equal(layer.forward(x[:1].expand(3, 512)), layer.forward(x[:1].repeat(3, 1)))  # row stride 0
    assert torch.equal(layer.forward(x[:1].expand(40, 512)), layer.forward(x[:1].repeat(40, 1)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [
    (12, 512, 136), (2, 16384, 40), (4, 8320, 33), (5, 8320, 33), (7, 6144, 8300), (13, 8320, 70), (13, 8192, 64), (70, 128, 1), (64, 8448, 1023),      # few rows; 64 x 64 tiles
    (512, 300, 2048), (513, 300, 2050), (700, 384, 2816), (2100, 8320, 1025), (1090, 256, 4097),  # the large tiles
])
def test_linear_tilings(hip_device, dtype, m, k, n):
    """Every split of the work, at its first and last rows, with more than 64 blocks
    of columns and an odd number of them."""
    x = _rand(m + k, m, k, dtype=dtype)
    wq, ws = _w8(n, n, k)
    _check_linear(x, wq, ws, _rand(n + 1, n, dtype=dtype))


@pytest.mark.parametrize("m", [2, 70])
def test_linear_quantised_input(hip_device, m):
    x = _rand(7, m, 1000, dtype=torch.bfloat16)
    wq, ws = _w8(8, 256, 1000)
    layer = Fp8Linear(wq, ws)
    y0 = layer.forward(x)
    assert torch.equal(layer.forward(quantize_rows_fp8(x), dtype=torch.bfloat16), y0)
    # scales that are no powers of two
    q, s = quantize_rows_fp8(x)
    s = s * torch.exp(_rand(9, *s.shape))
    got = _np(layer.forward((q, s), dtype=torch.float32))
    a, b = R.rows_value(_np(q.float()), _np(s)), R.weight_value(_np(wq.float()), _np(ws))
    tol = (1000 + 4 * 8) * U * (np.abs(a) @ np.abs(b).T) + U * np.abs(a @ b.T) + 1e-37
    assert (np.abs(got - a @ b.T) <= tol).all()


def test_linear_rows_are_apart(hip_device):
    """A row's non-finite values reach its own outputs alone, zero rows give
    the bias, and a row's result does not depend on its neighbours."""
    x = _rand(10, 50, 384, dtype=torch.bfloat16)
    wq, ws = _w8(11, 96, 384)
    bias = _rand(12, 96, dtype=torch.bfloat16)
    layer = Fp8Linear(wq, ws, bias)
    y0 = layer.forward(x)
    x2 = x.clone()
    x2[3, 7], x2[20, 200], x2[30] = float("nan"), float("inf"), 0
    y = layer.forward(x2)
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[20]).all())
    assert torch.equal(y[30], bias)
    same = [i for i in range(50) if i not in (3, 20, 30)]
    assert torch.equal(y[same], y0[same])


def test_linear_bias_of_another_type(hip_device):
    """A bias is read at the call, whatever its type and strides."""
    bias = _rand(21, 300, 2, dtype=torch.float32)[:, 0]
    was = bias.clone()
    layer = Fp8Linear(*_w8(22, 300, 256), bias)
    for m in (3, 40, 3000):
        x = _rand(m, m, 256, dtype=torch.bfloat16)
        y = layer.forward(x)
        bias.copy_(was + 64.0)
        moved = layer.forward(x)
        bias.copy_(was)
        # two roundings of the bias to bf16 and two of the result: 2^-8 of each
        tol = 2.0 ** -8 * (y.float().abs() + moved.float().abs() + was.abs() + (was + 64.0).abs()) + 1e-3
        assert bool(((moved.float() - y.float() - 64.0).abs() <= tol).all())
        assert torch.equal(layer.forward(x), y)


def test_linear_stream_and_graph(hip_device):
    x = _rand(13, 24, 512, dtype=torch.float16)
    wq, ws = _w8(14, 300, 512)
    layer = Fp8Linear(wq, ws)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = layer.forward(x)
    side.synchronize()
    assert torch.equal(got, layer.forward(x))
    big = _rand(15, 300, 512, dtype=torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap, cap_big = layer.forward(x), layer.forward(big)
    for seed in (16, 17, 18):
        x.copy_(_rand(seed, 24, 512, dtype=torch.float16))
        big.copy_(_rand(seed + 50, 300, 512, dtype=torch.float16))
        graph.replay()
        want, want_big = layer.forward(x), layer.forward(big)
        torch.cuda.synchronize()
        assert torch.equal(cap, want) and torch.equal(cap_big, want_big)


def test_linear_refusals(hip_device):
    wq, ws = _w8(1, 64, 256)
    x = _rand(1, 4, 256, dtype=torch.bfloat16)
    layer = Fp8Linear(wq, ws)
    for bad in (lambda: Fp8Linear(wq.float(), ws), lambda: Fp8Linear(wq, ws.double()), lambda: Fp8Linear(wq, ws[:, :1]),
                lambda: Fp8Linear(wq, ws, torch.zeros(63, device=hip_device)), lambda: Fp8Linear(wq[None], ws),
                lambda: layer.forward(x[:, :128]), lambda: layer.forward(x.double()),
                lambda: layer.forward(x, out=torch.empty(4, 65, dtype=torch.bfloat16, device=hip_device)),
                lambda: layer.forward(x, out=torch.empty(4, 64, device=hip_device)),
                lambda: layer.forward(x, out=torch.empty(64, 4, dtype=torch.bfloat16, device=hip_device).t()),
                lambda: layer.forward(quantize_rows_fp8(x)),
                lambda: layer.forward((x, ws), dtype=torch.bfloat16),
                lambda: quantize_rows_fp8(x[0]), lambda: quantize_rows_fp8(x[:, :0]),
                lambda: quantize_weight_fp8(x[0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        layer.forward(x.cpu())


# ------------------------------------------------------------------- experts
def _mlp_with_tol(x, w, dtype):
    """y of rows x in 64 bits, and how far a right kernel may be from it."""
    w1, s1, w3, s3, w2, s2 = w
    xv = R.rows_value(*R.quantize_rows(x))
    a, b, c = R.weight_value(w1, s1), R.weight_value(w3, s3), R.weight_value(w2, s2)
    h, inter = a.shape[1], a.shape[0]
    sums = lambda k: (k + 3 * (k // 128)) * U  # noqa: E731
    g, u = xv @ a.T, xv @ b.T
    eg, eu = sums(h) * (np.abs(xv) @ np.abs(a).T), sums(h) * (np.abs(xv) @ np.abs(b).T)
    silu = g / (1 + np.exp(-g))
    f = silu * u
    # |silu'| < 1.1; exp, reciprocal and two products: 2^-20 at most
    ef = (1.1 * eg + 2.0 ** -20 * np.abs(silu)) * (np.abs(u) + eu) + np.abs(silu) * eu
    q, s = R.quantize_rows(f)
    se = np.repeat(s, 128, 1)
    lo, _ = R.quantize_rows(f)
    # possible values of f^: rounding f - ef and f + ef on the block's scale, or,
    # where the block's largest may cross to the next scale, on that one
    top = np.abs(f).reshape(len(f), -1, 128)
    tmax, terr = top.max(2), ef.reshape(len(f), -1, 128).max(2)
    wobble = np.zeros_like(f)
    for sc in (R.pow2_scale(np.maximum(tmax - terr, 0)), R.pow2_scale(tmax + terr)):
        r = np.repeat(sc, 128, 1)
        for v in (f - ef, f + ef):
            wobble = np.maximum(wobble, np.abs(R.e4m3_round(np.clip(v / r, -448, 448)) * r - q * se))
    fv = q * se
    y = fv @ c.T
    tol = sums(inter) * (np.abs(fv) @ np.abs(c).T) + _truncated(fv, c) + wobble @ np.abs(c).T + 1e-37
    tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(y) + tol)
    return y, tol + (2.0 ** -25 if dtype == torch.float16 else 0)


def _weights(seed, e, h, inter):
    return (*_w8(seed, e, inter, h), *_w8(seed + 1, e, inter, h), *_w8(seed + 2, e, h, inter))


def _check_experts(x, ids, mask, w, slots=None, ids_arg=None):
    n, k = ids.shape
    if slots is None:
        slots = torch.full((n, k, x.shape[1]), 7.0, dtype=x.dtype, device=x.device)
    before = slots.clone()
    ex = Fp8GroupedExperts(*w)
    got = ex.forward(x, ids if ids_arg is None else ids_arg, mask, slots)
    assert got is slots
    m = mask[:, None].expand(n, k) if mask.dim() == 1 else mask
    wn = [_np(t.float()) for t in w]
    take = (m != 0) & (ids >= 0) & (ids < w[0].shape[0])
    assert torch.equal(slots[~take], before[~take])
    for e in range(w[0].shape[0]):
        b, s = torch.nonzero(take & (ids == e), as_tuple=True)
        if b.numel() == 0:
            continue
        y, tol = _mlp_with_tol(_np(x[b]), [t[e] for t in wn], x.dtype)
        d = np.abs(_np(slots[b, s]) - y)
        assert (d <= tol).all(), (e, float((d / tol).max()), int((d > tol).sum()))
        # and as a whole near it
        assert np.linalg.norm(d) <= (torch.finfo(x.dtype).eps + 2e-3) * np.linalg.norm(y)
    return ex, slots


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k,e,h,inter", [
    (1, 8, 16, 256, 128), (1, 1, 1, 128, 128), (5, 2, 3, 384, 256), (32, 8, 64, 256, 384), (64, 6, 8, 256, 128),
    (128, 8, 8, 256, 256), (200, 6, 8, 256, 384), (700, 4, 5, 384, 128), (1500, 2, 40, 128, 256), (90, 12, 200, 128, 128),
])
def test_experts(hip_device, dtype, n, k, e, h, inter):
    x = _rand(n + h, n, h, dtype=dtype)
    g = torch.Generator().manual_seed(n)
    ids = torch.stack([torch.randperm(max(e, k), generator=g)[:k] for _ in range(n)]).to(hip_device)  # some past e
    mask = (torch.rand(n, k, generator=g) < 0.7).to(hip_device)
    _check_experts(x, ids, mask, _weights(n + 1, e, h, inter))


@pytest.mark.parametrize("n,h,inter", [(6, 2048, 768), (40, 2560, 1536), (150, 2048, 768)])
def test_experts_family_shapes(hip_device, n, h, inter):
    e, k = 4, 2
    x = _rand(n, n, h, dtype=torch.bfloat16)
    ids = torch.randint(0, e, (n, k), generator=torch.Generator().manual_seed(n)).to(hip_device)  # an expert twice
    _check_experts(x, ids, torch.ones(n, dtype=torch.bool, device=hip_device), _weights(n, e, h, inter))


@pytest.mark.parametrize("n", [20, 600])
def test_experts_uneven_and_masks(hip_device, n):
    e, k, h, inter = 8, 3, 256, 128
    x = _rand(n, n, h, dtype=torch.bfloat16)
    w = _weights(3, e, h, inter)
    ids = torch.full((n, k), 5, device=hip_device)          # every row on one expert, three times
    _check_experts(x, ids, torch.ones(n, dtype=torch.bool, device=hip_device), w)
    ids[::2, 1], ids[1::2, 2], ids[0, 0] = -1, 8, 1 << 40   # out of range: not taken
    flags = (torch.arange(n, device=hip_device) % 3 != 0)
    _check_experts(x, ids, flags, w)
    _check_experts(x, ids, torch.zeros(n, k, dtype=torch.bool, device=hip_device), w)      # nothing
    m = torch.zeros(n, 2 * k, dtype=torch.bool, device=hip_device)
    m[:, ::2] = flags[:, None]
    _check_experts(x, ids, m[:, ::2], w)                    # a strided mask
    wide = torch.zeros(n, 9, dtype=torch.long, device=hip_device)
    wide[:, 2:5] = ids
    _check_experts(x, wide[:, 2:5], flags, w)               # strided ids
    _check_experts(x, ids, flags, w, ids_arg=ids.clamp(-1, 100).int())
    big = torch.full((n, k + 1, h + 8), 7.0, dtype=torch.bfloat16, device=hip_device)
    _check_experts(x, ids, flags, w, slots=big[:, 1:, :h])  # strided slots
    assert bool((big[:, 0] == 7).all()) and bool((big[:, :, h:] == 7).all())
    xw = torch.zeros(n, h + 24, dtype=torch.bfloat16, device=hip_device)
    xw[:, 8:8 + h] = x
    _check_experts(xw[:, 8:8 + h], ids, flags, w)           # strided rows


@pytest.mark.parametrize("n", [30, 700])
def test_experts_scales_far_apart(hip_device, n):
    """Blocks scaled by 0, by 2^-60 of their neighbours, by a negative number."""
    e, k, h, inter = 5, 3, 512, 256
    x = _rand(n, n, h, dtype=torch.bfloat16)
    w = list(_weights(6, e, h, inter))
    w[1][0, 0, 1] = 0.0
    w[3][1, 1, 2] = 2.0 ** -60
    w[1][2, :, 0] = 2.0 ** -70
    w[3][3, 0, :] *= -1.0
    w[5][0, 1, 1], w[5][1, 0, 0] = 0.0, -1e-3
    ids = torch.stack([torch.randperm(e, generator=torch.Generator().manual_seed(i))[:k] for i in range(n)]).to(hip_device)
    _check_experts(x, ids, torch.ones(n, dtype=torch.bool, device=hip_device), tuple(w))


@pytest.mark.parametrize("k", [1, 5, 8])
def test_experts_of_one_token(hip_device, k):
    """One token: an expert in several slots, ids out of range, masked slots, as many
    slots as experts."""
    e, h, inter = 5, 384, 256
    x = _rand(k, 1, h, dtype=torch.bfloat16)
    ids = torch.tensor([[3, 3, -1, 5, 0, 3, 1, 2][:k]], device=hip_device)
    _check_experts(x, ids, torch.ones(1, dtype=torch.bool, device=hip_device), _weights(8, e, h, inter))
    flags = torch.tensor([[1, 0, 1, 1, 1, 1, 0, 1][:k]], dtype=torch.bool, device=hip_device)
    _check_experts(x, ids, flags, _weights(8, e, h, inter))
    _check_experts(x, ids, torch.zeros(1, dtype=torch.bool, device=hip_device), _weights(8, e, h, inter))


@pytest.mark.parametrize("n", [7, 600])
def test_experts_one_row_of_ids_for_all(hip_device, n):
    """ids and masks of row stride 0."""
    e, k, h, inter = 6, 3, 256, 128
    w = _weights(9, e, h, inter)
    x = _rand(n, n, h, dtype=torch.bfloat16)
    ids = torch.tensor([[4, 0, 2]], device=hip_device).expand(n, k)
    flags = torch.tensor([[1, 1, 0]], dtype=torch.uint8, device=hip_device).expand(n, k)
    _, one = _check_experts(x, ids, flags, w)
    _, two = _check_experts(x, ids.contiguous(), flags.contiguous().bool(), w)
    assert torch.equal(one, two)
    _check_experts(x[:1].expand(n, h), ids, torch.ones(1, dtype=torch.bool, device=hip_device).expand(n), w)


def test_experts_rows_do_not_depend_on_others(hip_device):
    """Two calls give the same bits, and so does another order of the tokens."""
    n, k, e, h, inter = 90, 4, 6, 256, 256
    x = _rand(2, n, h, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, e, (n, k), generator=g).to(hip_device)
    mask = torch.ones(n, dtype=torch.bool, device=hip_device)
    ex = Fp8GroupedExperts(*_weights(9, e, h, inter))
    out = [torch.zeros(n, k, h, dtype=torch.bfloat16, device=hip_device) for _ in range(3)]
    ex.forward(x, ids, mask, out[0])
    ex.forward(x, ids, mask, out[1])
    p = torch.randperm(n, generator=g).to(hip_device)
    ex.forward(x[p], ids[p], mask, out[2])
    assert torch.equal(out[0], out[1]) and torch.equal(out[0][p], out[2])


@pytest.mark.parametrize("n", [3, 500])
def test_experts_streams_and_graphs(hip_device, n):
    """A captured call replayed beside eager ones and another captured call of
    the same experts: no scratch is shared."""
    k, e, h, inter = 4, 6, 256, 128
    ex = Fp8GroupedExperts(*_weights(4, e, h, inter))
    mk = lambda seed: (_rand(seed, n, h, dtype=torch.float16),  # noqa: E731
                       torch.randint(0, e, (n, k), generator=torch.Generator().manual_seed(seed)).to(hip_device))
    mask = torch.ones(n, dtype=torch.bool, device=hip_device)
    zero = lambda: torch.zeros(n, k, h, dtype=torch.float16, device=hip_device)  # noqa: E731
    (xa, ia), (xb, ib) = mk(1), mk(2)
    oa, ob = zero(), zero()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        ex.forward(xa, ia, mask, oa)
    with torch.cuda.graph(gb):
        ex.forward(xb, ib, mask, ob)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for seed in (3, 4, 5):
        x2, i2 = mk(seed)
        xa.copy_(x2)
        ia.copy_(i2)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            ga.replay()
        with torch.cuda.stream(s2):
            gb.replay()
        eager = ex.forward(x2, i2, mask, zero())
        want_b = ex.forward(xb, ib, mask, zero())
        torch.cuda.synchronize()
        assert torch.equal(oa, eager) and torch.equal(ob, want_b)


def test_experts_refusals(hip_device):
    w = _weights(1, 4, 256, 128)
    ex = Fp8GroupedExperts(*w)
    x = _rand(1, 4, 256, dtype=torch.bfloat16)
    ids = torch.zeros(4, 2, dtype=torch.long, device=hip_device)
    mask = torch.ones(4, dtype=torch.bool, device=hip_device)
    out = torch.zeros(4, 2, 256, dtype=torch.bfloat16, device=hip_device)
    pad = torch.zeros(4, 2, 257, dtype=torch.bfloat16, device=hip_device)
    for bad in (lambda: ex.forward(x.float(), ids, mask, out.float()), lambda: ex.forward(x, ids, mask, out.half()),
                lambda: ex.forward(x[:, :128], ids, mask, out), lambda: ex.forward(x, ids, mask[:3], out),
                lambda: ex.forward(x, ids, mask, out[:, :1]), lambda: ex.forward(x, ids, mask, pad[:, :, :256]),
                lambda: ex.forward(x, ids, mask, pad[:, :, 1:]), lambda: Fp8GroupedExperts(*w[:4], w[0], w[1]),
                lambda: Fp8GroupedExperts(w[0], w[1][:, :, :1], *w[2:]), lambda: Fp8GroupedExperts(*_weights(1, 2, 256, 64)),
                lambda: Fp8GroupedExperts(w[0].float(), *w[1:]), lambda: Fp8SharedExperts(*w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ex.forward(x.cpu(), ids, mask, out)
    assert ex.forward(x[:0], ids[:0], mask[:0], out[:0]).shape == (0, 2, 256)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,h,inter", [(1, 2560, 1536), (7, 256, 128), (40, 384, 256), (300, 256, 384), (1030, 128, 256)])
def test_shared_experts(hip_device, dtype, m, h, inter):
    x, add = _rand(m, m, h, dtype=dtype), _rand(m + 1, m, h, dtype=dtype)
    w = [t[0] for t in _weights(m, 1, h, inter)]
    sh = Fp8SharedExperts(*w)
    y, tol = _mlp_with_tol(_np(x), [_np(t.float()) for t in w], dtype)
    d = np.abs(_np(sh.forward(x)) - y)
    assert (d <= tol).all(), float((d / tol).max())
    got = sh.forward(x, addend=add)
    want = y + _np(add)
    d = np.abs(_np(got) - want)
    assert (d <= tol + torch.finfo(dtype).eps / 2 * np.abs(want)).all()
    wide = torch.full((m, h + 8), 7.0, dtype=dtype, device=hip_device)
    assert torch.equal(sh.forward(x, out=wide[:, :h], addend=add), got) and bool((wide[:, h:] == 7).all())
    assert sh.forward(x[:0]).shape == (0, h)


def test_quantised_from_float_weights(hip_device):
    """from_weights is the quantiser followed by the 8-bit experts."""
    e, h, inter, n, k = 3, 256, 128, 10, 2
    w1, w3 = _rand(1, e, inter, h, scale=0.05), _rand(2, e, inter, h, scale=0.05)
    w2 = _rand(3, e, h, inter, scale=0.05)
    x = _rand(4, n, h, dtype=torch.bfloat16)
    ids = torch.randint(0, e, (n, k), generator=torch.Generator().manual_seed(1)).to(hip_device)
    mask = torch.ones(n, dtype=torch.bool, device=hip_device)
    a = Fp8GroupedExperts.from_weights(w1, w3, w2)
    b = Fp8GroupedExperts(*quantize_weight_fp8(w1), *quantize_weight_fp8(w3), *quantize_weight_fp8(w2))
    out = [torch.zeros(n, k, h, dtype=torch.bfloat16, device=hip_device) for _ in range(2)]
    assert torch.equal(a.forward(x, ids, mask, out[0]), b.forward(x, ids, mask, out[1]))
    l1, l2 = Fp8Linear.from_weight(w1[0]), Fp8Linear(*quantize_weight_fp8(w1[0]))
    assert torch.equal(l1.forward(x), l2.forward(x))


@pytest.mark.parametrize("h,inter", [(384, 256), (256, 128)])
def test_experts_one_row_of_any_stride(hip_device, h, inter):
    """The row stride of a single row means nothing: it may be odd, or 0."""
    e, k = 4, 3
    w = _weights(5, e, h, inter)
    sh = Fp8SharedExperts(*(t[0] for t in w))
    row = _rand(1, 1, h, dtype=torch.bfloat16)
    ids = torch.tensor([[2, 0, 3]], device=hip_device)
    flag = torch.ones(1, dtype=torch.bool, device=hip_device)
    _, want = _check_experts(row, ids, flag, w)
    dense = sh.forward(row, addend=row)
    odd = torch.zeros(1, h + 3, dtype=torch.bfloat16, device=hip_device)
    odd[:, :h] = row
    for x in (odd[:, :h], row[0].expand(1, h), row.as_strided((1, h), (1, 1))):
        _, got = _check_experts(x, ids, flag, w)
        assert torch.equal(got, want)
        assert torch.equal(sh.forward(x, addend=x), dense)
    out = torch.zeros(1, h + 3, dtype=torch.bfloat16, device=hip_device)
    sh.forward(row, out=out[:, :h], addend=odd[:, :h])
    assert torch.equal(out[:, :h], dense) and bool((out[:, h:] == 0).all())
    slots = torch.zeros(1, k * h + 5, dtype=torch.bfloat16, device=hip_device)
    _check_experts(row, ids, flag, w, slots=slots[:, :k * h].view(1, k, h))
    assert bool((slots[:, k * h:] == 0).all())


def test_experts_overlapping_slots_are_refused(hip_device):
    """Slots that lie on each other have no defined result."""
    n, k, e, h = 4, 2, 3, 256
    ex = Fp8GroupedExperts(*_weights(1, e, h, 128))
    x = _rand(1, n, h, dtype=torch.bfloat16)
    ids = torch.zeros(n, k, dtype=torch.long, device=hip_device)
    mask = torch.ones(n, dtype=torch.bool, device=hip_device)
    mem = torch.zeros(n * k * h, dtype=torch.bfloat16, device=hip_device)
    for strides in ((0, h), (k * h, 0), (h, h), (8, n * h), (k * h, 8)):
        with pytest.raises(ValueError):
            ex.forward(x, ids, mask, mem.as_strided((n, k, h), (*strides, 1)))
    assert not bool(mem.any())
    _check_experts(x, ids, mask, _weights(1, e, h, 128), slots=mem.view(k, n, h).transpose(0, 1))


def test_linear_quantised_rows_end_inside_their_storage(hip_device):
    """A row of 8-bit x is read up to its whole last block: where that is not there,
    the call is refused."""
    x = _rand(3, 5, 200, dtype=torch.bfloat16)
    wq, ws = _w8(4, 64, 200)
    layer = Fp8Linear(wq, ws)
    q, s = quantize_rows_fp8(x)
    want = layer.forward((q, s), dtype=torch.bfloat16)
    short = torch.zeros(4 * 256 + 200, dtype=torch.uint8, device=hip_device)
    short[:] = torch.as_strided(q.view(torch.uint8), (4 * 256 + 200,), (1,))
    with pytest.raises(ValueError):
        layer.forward((short.view(torch.float8_e4m3fn).as_strided((5, 200), (256, 1)), s), dtype=torch.bfloat16)
    assert torch.equal(layer.forward((q[2:], s[2:]), dtype=torch.bfloat16), want[2:])
    assert torch.equal(layer.forward((q[:4], s[:4]), dtype=torch.bfloat16), want[:4])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(8, 2048, 1000), (40, 2048, 520), (200, 1000, 300), (520, 256, 2050)])
def test_linear_as_a_whole(hip_device, dtype, m, k, n):
    """The norm of all errors, in every plan: the roundings of the outputs, half a step
    of each at most; what the 8-bit instructions drop, whose signs are those of the
    products dropped from, so the squares add up (7 of 8 products, 2^-13 of the
    largest each); K roundings of sums in fp32, likewise."""
    x = _rand(m + 3, m, k, dtype=dtype)
    wq, ws = _w8(n + 3, n, k)
    y = R.linear(_np(x), _np(wq.float()), _np(ws))
    xv, wv = np.abs(R.rows_value(*R.quantize_rows(_np(x)))), np.abs(R.weight_value(_np(wq.float()), _np(ws)))
    dropped = 0.0
    for k0 in range(0, k, 8):
        top = np.zeros_like(y)
        for i in range(k0, min(k0 + 8, k)):
            np.maximum(top, np.multiply.outer(xv[:, i], wv[:, i]), out=top)
        dropped += 7 * (2.0 ** -13 * np.linalg.norm(top)) ** 2
    tol = torch.finfo(dtype).eps / 2 * np.linalg.norm(y) + np.sqrt(dropped) + np.sqrt(k) * U * np.linalg.norm(xv @ wv.T)
    assert tol < 0.005 * np.linalg.norm(y)
    got = _np(Fp8Linear(wq, ws).forward(x))
    assert np.linalg.norm(got - y) <= tol, np.linalg.norm(got - y) / np.linalg.norm(y)


@pytest.mark.parametrize("n,k,e,h,inter", [(9001, 2, 20, 256, 128), (1300, 12, 24, 128, 256), (900, 6, 300, 128, 128)])
def test_experts_grouped_by_one_workgroup(hip_device, n, k, e, h, inter):
    """More than 8192 tokens, 8 slots or 256 experts: another grouping."""
    x = _rand(n, n, h, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, e, (n, k), generator=g).to(hip_device)
    mask = (torch.rand(n, generator=g) < 0.5).to(hip_device)
    w = _weights(n, e, h, inter)
    _, slots = _check_experts(x, ids, mask, w)
    of = (ids == 3) & mask[:, None]
    b, s = torch.nonzero(of, as_tuple=True)
    y = R.mlp(_np(x[b]), *(_np(t[3].float()) for t in w))
    assert np.linalg.norm(_np(slots[b, s]) - y) <= (torch.finfo(x.dtype).eps + 2e-3) * np.linalg.norm(y)


@pytest.mark.parametrize("m,k,n", [(8, 2048, 4096), (12, 4096, 2048), (64, 1024, 2048), (333, 1000, 1111),
                                   (4096, 1024, 512)])
def test_linear_gives_the_same_bits_again(hip_device, m, k, n):
    """The same call twice, beside other work: bit for bit, and so on the quantised rows."""
    for dtype in (torch.bfloat16, torch.float32):
        x = _rand(m, m, k, dtype=dtype)
        layer = Fp8Linear(*_w8(n, n, k), _rand(1, n, dtype=dtype))
        want = layer.forward(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [layer.forward(x) for _ in range(3)]
        again = [layer.forward(x) for _ in range(3)] + [layer.forward(quantize_rows_fp8(x), dtype=dtype)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in other + again)


@pytest.mark.parametrize("n,e,k,h,inter", [(1, 128, 8, 2048, 768), (32, 128, 8, 2048, 768), (300, 16, 6, 2048, 768)])
def test_experts_give_the_same_bits_again(hip_device, n, e, k, h, inter):
    """The same call twice, beside other work, bit for bit (rows find their places in
    their expert's list in any order)."""
    x = _rand(n, n, h, dtype=torch.bfloat16)
    ids = torch.randint(0, e, (n, k), generator=torch.Generator().manual_seed(n)).to(hip_device)
    mask = torch.ones(n, dtype=torch.bool, device=hip_device)
    q = lambda *s: ((90 * torch.randn(*s, device=hip_device)).clamp(-448, 448).to(torch.float8_e4m3fn),  # noqa: E731
                    torch.full((s[0], s[1] // 128, s[2] // 128), 2e-4, device=hip_device))
    ex = Fp8GroupedExperts(*q(e, inter, h), *q(e, inter, h), *q(e, h, inter))
    zero = lambda: torch.zeros(n, k, h, dtype=torch.bfloat16, device=hip_device)  # noqa: E731
    want = ex.forward(x, ids, mask, zero())
    slots = [zero() for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ex.forward(x, ids, mask, slots[0])
        ex.forward(x, ids, mask, slots[1])
    ex.forward(x, ids, mask, slots[2])
    ex.forward(x, ids, mask, slots[3])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in slots)

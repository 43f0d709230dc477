"""Rotation by positions of several axes, the 8-bit cache, attention and
importance over it, against their definitions in 64 bits."""

import math

import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------ rotation
def rotate_ref(x, positions, inv, sections, interleaved, adjacent, inverse):
    y, half, sizes = x.double().clone(), inv.shape[0], torch.zeros_like(x, dtype=torch.float64)
    a_n = len(sections)
    for i in range(half):
        if interleaved:
            a = i % a_n if i < a_n * sections[i % a_n] else 0
        else:
            a = next(j for j in range(a_n) if i < sum(sections[:j + 1]))
        ang = positions[a].double() * float(inv[i])
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None] * (-1 if inverse else 1)
        lo, hi = (2 * i, 2 * i + 1) if adjacent else (i, half + i)
        u, w = x[..., lo].double(), x[..., hi].double()
        y[..., lo], y[..., hi] = u * c - w * s, w * c + u * s
        sizes[..., lo] = sizes[..., hi] = u.abs() + w.abs()
    return y, sizes


def rotate_close(got, want, sizes, turned):
    """Sine and cosine: half a turn's fraction is rounded by 2^-25 (pi 2^-25 of angle), they themselves by at most
    two steps of 2^-23, product and sum by three half steps of 2^-24: under 6e-7 of |x1| + |x2|.  Then one rounding."""
    dt = got.dtype
    tol = 6e-7 * sizes + (half_step(dt) if dt != F32 else 0.0) * (want.abs() + 6e-7 * sizes)
    tol += 2.0 ** -25 if dt == F16 else 0.0  # its subnormals
    assert bool(((got.cpu().double() - want).abs() <= tol)[..., :turned].all())
    assert torch.equal(got.cpu().double()[..., turned:], want[..., turned:])


@pytest.mark.parametrize("n,h,kv,d,turned,sections,interleaved,adjacent,inverse,dt", [
    (1, 32, 4, 128, 128, (24, 20, 20), True, False, False, BF16),
    (7, 32, 4, 128, 128, (16, 24, 24), False, False, True, F16),
    (33, 3, 1, 64, 64, (32,), False, True, False, F32),
    (5, 2, 2, 256, 128, (31, 0, 33), False, False, False, F32),
    (9, 4, 2, 192, 64, (10, 11, 11), True, True, True, BF16),
    (130, 5, 5, 72, 40, (9, 11), True, False, False, F16),     # no multiple of 8
    (6, 2, 1, 1024, 1024, (200, 100, 100, 112), True, False, False, F32),
    (3, 1, 1, 2, 2, (1,), False, True, False, F32),
])
def test_rotate(hip_device, n, h, kv, d, turned, sections, interleaved, adjacent, inverse, dt):
    from table_moe.ops import rotate_positions

    g = torch.Generator().manual_seed(n * d + h)
    q, k = torch.randn(n, h, d, generator=g).to(dt), torch.randn(n, kv, d, generator=g).to(dt)
    pos = torch.randint(-1000, 300000, (len(sections), n), generator=g)
    inv = (1e6 ** (-torch.arange(turned // 2).double() / (turned // 2))).float()
    dev = hip_device
    qo, ko = rotate_positions(q.to(dev), k.to(dev), pos.to(dev), inv.to(dev), sections, interleaved=interleaved,
                              adjacent=adjacent, inverse=inverse)
    for x, y in ((q, qo), (k, ko)):
        assert y.dtype == dt and y.shape == x.shape
        rotate_close(y, *rotate_ref(x, pos, inv, sections, interleaved, adjacent, inverse), turned)
    # without keys; positions in 32 bits; a single axis as one row
    q1, none = rotate_positions(q.to(dev), None, pos.to(dev).int(), inv.to(dev), sections, interleaved=interleaved,
                                adjacent=adjacent, inverse=inverse)
    assert none is None and torch.equal(q1, qo)


def test_rotate_views_in_place_and_streams(hip_device):
    """q and k as views of one fused projection, written in place; heads before tokens; empty; another stream."""
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(5)
    n, h, kv, d = 37, 8, 2, 128
    fused = torch.randn(n, (h + 2 * kv) * d, generator=g).to(BF16)
    pos = torch.randint(0, 9000, (3, n), generator=g)
    inv = (1e6 ** (-torch.arange(64).double() / 64)).float()
    sec = (24, 20, 20)
    f = fused.to(dev)
    q, k = f[:, :h * d].view(n, h, d), f[:, h * d:(h + kv) * d].view(n, kv, d)
    want_q, want_k = rotate_positions(q, k, pos.to(dev), inv.to(dev), sec, interleaved=True)
    rotate_close(want_q, *rotate_ref(fused[:, :h * d].view(n, h, d), pos, inv, sec, True, False, False), 128)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, b = rotate_positions(by_head, k, pos.to(dev), inv.to(dev), sec, interleaved=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, want_q) and torch.equal(b, want_k)
    rest = f[:, (h + kv) * d:].clone()
    r = rotate_positions(q, k, pos.to(dev), inv.to(dev), sec, interleaved=True, out=(q, k))
    assert r[0] is q and torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(f[:, (h + kv) * d:], rest)
    # turned back: two roundings of a half step each, and the rotation keeps a pair's length
    back, _ = rotate_positions(want_q, want_k, pos.to(dev), inv.to(dev), sec, interleaved=True, inverse=True)
    x = fused[:, :h * d].view(n, h, d).float()
    length = torch.hypot(x[..., :64], x[..., 64:]).repeat(1, 1, 2)
    assert bool(((back.cpu().float() - x).abs() <= 3.5 * half_step(BF16) * length).all())
    e, ek = rotate_positions(q[:0], k[:0], pos[:, :0].to(dev), inv.to(dev), sec)
    assert e.shape == (0, h, d) and ek.shape == (0, kv, d)


def test_rotate_gradients(hip_device):
    """Against the formula's transpose and against differences; second order; only one of q and k."""
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(6)
    n, h, kv, d, sec = 11, 3, 1, 64, (12, 10, 10)
    pos = torch.randint(0, 5000, (3, n), generator=g)
    inv = (1e4 ** (-torch.arange(32).double() / 32)).float()
    x, y = torch.randn(n, h, d, generator=g), torch.randn(n, kv, d, generator=g)
    wq, wk = torch.randn(n, h, d, generator=g), torch.randn(n, kv, d, generator=g)
    q, k = x.to(dev).requires_grad_(), y.to(dev).requires_grad_()
    args = (pos.to(dev), inv.to(dev), sec)
    qo, ko = rotate_positions(q, k, *args, interleaved=True)
    dq, dk = torch.autograd.grad((qo * wq.to(dev)).sum() + (ko * wk.to(dev)).sum(), (q, k))
    rotate_close(dq, *rotate_ref(wq, pos, inv, sec, True, False, True), d)
    rotate_close(dk, *rotate_ref(wk, pos, inv, sec, True, False, True), d)
    # the map is linear: a step of any size gives its derivative, up to the roundings of the two values
    step = torch.randn(n, h, d, generator=g)
    with torch.no_grad():
        q2, _ = rotate_positions((x + step).to(dev), y.to(dev), *args, interleaved=True)
    diff = ((q2 - qo).double() * wq.to(dev).double()).sum()
    assert abs(float(diff - (dq.double() * step.to(dev).double()).sum())) < 1e-5 * float((wq.abs() * (x.abs() + step.abs() + 1)).sum())
    only, = torch.autograd.grad(rotate_positions(x.to(dev), k, *args, interleaved=True)[1].sum(), k)
    rotate_close(only, *rotate_ref(torch.ones_like(y), pos, inv, sec, True, False, True), d)
    o, _ = rotate_positions(q, None, *args)
    first, = torch.autograd.grad((o ** 3).sum(), q, create_graph=True)
    second, = torch.autograd.grad(first.sum(), q)
    assert bool(torch.isfinite(second).all()) and float(second.abs().max()) > 0
    with torch.no_grad():
        assert not rotate_positions(q, k, *args)[0].requires_grad


def test_rotate_gradients_captured(hip_device):
    """Forward and gradient in one captured graph, replayed over other inputs between eager work."""
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(16)
    n, h, kv, d = 13, 4, 2, 64
    mk = lambda heads: torch.randn(n, heads, d, generator=g).to(BF16).to(dev)  # noqa: E731
    inv = (1e4 ** (-torch.arange(32).double() / 32)).float().to(dev)
    pos = torch.randint(0, 9000, (3, n), generator=g).to(dev)
    q, k, wq, wk = mk(h), mk(kv), mk(h), mk(kv)

    def step(q, k, wq, wk, pos):
        a, b = q.detach().requires_grad_(), k.detach().requires_grad_()
        y, z = rotate_positions(a, b, pos, inv, (12, 10, 10), interleaved=True)
        return y.detach(), z.detach(), *torch.autograd.grad((y, z), (a, b), (wq, wk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, wq, wk, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, wq, wk, pos)
    for _ in range(4):
        q.copy_(mk(h)), k.copy_(mk(kv)), wq.copy_(mk(h)), wk.copy_(mk(kv))
        pos.copy_(torch.randint(0, 9000, (3, n), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(q.clone(), k.clone(), wq, wk, pos)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rotate_refusals(hip_device):
    from table_moe.ops import rotate_positions

    dev = hip_device
    q, k = torch.zeros(4, 2, 64, device=dev), torch.zeros(4, 1, 64, device=dev)
    pos, inv = torch.zeros(3, 4, dtype=torch.long, device=dev), torch.ones(32, device=dev)
    ok = dict(q=q, k=k, positions=pos, inv_freq=inv, sections=(10, 11, 11))
    rotate_positions(**ok)
    buf = torch.zeros(9, 2, 64, device=dev)
    for kw in (dict(q=q[0]), dict(k=k[:3]), dict(k=k.half()), dict(k=torch.zeros(4, 1, 32, device=dev)),
               dict(q=q.double(), k=k.double()), dict(positions=pos[:, :3]), dict(positions=pos.float()),
               dict(sections=(10, 11)), dict(sections=(10, 11, 12)), dict(sections=(43, -11, 0)), dict(sections=None),
               dict(inv_freq=inv.double()), dict(inv_freq=torch.ones(33, device=dev), sections=(11, 11, 11)),
               dict(out=(q, None)), dict(out=(q[:, :1], k)), dict(out=(torch.zeros(4, 2, 64, device=dev, dtype=F16), k)),
               dict(q=buf[:4], out=(buf[2:6], k)), dict(out=(buf[:1].expand(4, 2, 64), k)),
               dict(positions=torch.zeros(5, 4, dtype=torch.long, device=dev), sections=(8, 8, 8, 4, 4)),
               dict(q=q.clone().requires_grad_(), out=(torch.empty_like(q), k))):
        with pytest.raises(ValueError):
            rotate_positions(**{**ok, **kw})
    with pytest.raises(RuntimeError):
        rotate_positions(q.cpu(), None, pos, inv, (10, 11, 11))


def test_rotate_outputs_that_overlap(hip_device):
    """Outputs may be their inputs, or other columns of the same rows; not each other's, nor the other's input."""
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(12)
    n, d = 9, 64
    fused = torch.randn(n, 8 * d, generator=g).to(dev)
    part = lambda a, b: fused[:, a * d:b * d].view(n, b - a, d)  # noqa: E731
    pos, inv = torch.arange(n, device=dev), torch.rand(d // 2, generator=g).to(dev)
    q, k = part(0, 2), part(2, 4)
    want = rotate_positions(q, k, pos, inv)
    got = rotate_positions(q, k, pos, inv, out=(part(4, 6), part(6, 8)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[0], part(4, 6))
    one = torch.zeros(n, 2, d, device=dev)
    for out in ((k, q), (one, one), (part(2, 4), part(6, 8)), (part(4, 6), part(5, 7)), (part(1, 3), part(6, 8)),
                (one, fused.view(-1)[d:d + n * 2 * d].view(n, 2, d))):
        with pytest.raises(ValueError, match="overlap"):
            rotate_positions(q, k, pos, inv, out=out)
    with pytest.raises(ValueError, match="overlap"):  # one tensor as both inputs, turned twice in place
        rotate_positions(one, one, pos, inv, out=(one, one))
    rotate_positions(one, one, pos, inv)


def test_outputs_that_a_graph_has_saved(hip_device):
    """A write to a tensor that a backward needs is an error there, as after torch's own writes in place."""
    from table_moe.ops import Fp8KVCache, rotate_positions

    dev = hip_device
    q = torch.randn(3, 2, 64, device=dev)
    w = torch.ones(3, 2, 64, device=dev, requires_grad=True)
    pos, inv = torch.arange(3, device=dev), torch.ones(32, device=dev)
    y = (q * w).sum()
    rotate_positions(q, None, pos, inv, out=(q, None))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    cache = Fp8KVCache(1, 1, 64, device=dev)
    table, one = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    out = torch.ones(1, 1, 64, dtype=F16, device=dev)
    v = torch.ones(1, 1, 64, dtype=F16, device=dev, requires_grad=True)
    y = (out * v).sum()
    cache.attend(torch.ones(1, 1, 64, dtype=F16, device=dev), table, one, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():
        r = torch.ones(3, 2, 64, device=dev)
        rotate_positions(r, None, pos, inv, out=(r, None))
    with pytest.raises(ValueError, match="gradient"):
        rotate_positions(w, None, pos, inv.clone().requires_grad_())


# --------------------------------------------------------------------- append
def filled(g, pages, kv, page, d, dv, dev):
    """A cache in use: (Fp8KVCache, plain cells and scales of K and V)."""
    from table_moe.ops import Fp8KVCache

    cache = Fp8KVCache(pages, kv, d, dv, page, device=dev)
    plain = []
    for which, cols in ((0, d), (1, dv)):
        x = torch.randn(pages, kv, page, cols, generator=g).double() * torch.exp(torch.randn(pages, kv, 1, 1, generator=g).double())
        s = torch.tensor([[R.scale_of(float(x[p, h].abs().max())) for h in range(kv)] for p in range(pages)]).double()
        c = R.e4m3(x / s[:, :, None, None])
        (cache.v if which else cache.k).view(torch.uint8).copy_(R.pack(c, bool(which)).view(torch.uint8))
        (cache.v_scale if which else cache.k_scale).copy_(s.float())
        plain += [c, s]
    return cache, plain


def same_cells(packed, want, values):
    got = R.raw(packed, values)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def table_of(g, counts, most, pages):
    t = torch.randperm(pages, generator=g)[:sum(counts)].to(torch.int32)
    out, at = torch.full((len(counts), most), -1, dtype=torch.int32), 0
    for b, c in enumerate(counts):
        out[b, :c] = t[at:at + c]
        at += c
    return out


@pytest.mark.parametrize("page,d,dv,kv,lens,new,dt", [
    (64, 128, 128, 4, [1, 64, 65, 200], None, BF16),            # one token each: begun and partly full pages
    (32, 64, 64, 2, [33, 5, 97, 64], [33, 2, 40, 0], F16),       # whole pages, odd ends, none
    (128, 192, 128, 3, [300, 129, 128], [171, 1, 128], F32),
    (64, 256, 256, 1, [190, 70], [100, 3], BF16),
    (128, 192, 192, 1, [257], [257], F16),
])
def test_append(hip_device, page, d, dv, kv, lens, new, dt):
    g = torch.Generator().manual_seed(page + d + len(lens))
    n = len(lens) if new is None else sum(new)
    counts = [-(-x // page) for x in lens]
    cache, (kc, ks, vc, vs) = filled(g, sum(counts) + 2, kv, page, d, dv, hip_device)
    table = table_of(g, counts, max(counts) + 1, sum(counts) + 2)
    starts = None if new is None else torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    # sizes over a wide range: some scales rise, some do not
    k = (torch.randn(n, kv, d, generator=g) * torch.exp(1.5 * torch.randn(n, kv, 1, generator=g))).to(dt)
    v = (torch.randn(n, kv, dv, generator=g) * torch.exp(1.5 * torch.randn(n, kv, 1, generator=g))).to(dt)
    lengths = torch.tensor(lens, dtype=torch.int32)
    dev = hip_device
    for _ in range(2):  # the same call again changes nothing more
        cache.append(k.to(dev), v.to(dev), table.to(dev), lengths.to(dev), None if starts is None else starts.to(dev))
        for rows, c, s in ((k, kc, ks), (v, vc, vs)):
            R.append(c, s, rows, table, lengths, starts)
        assert torch.equal(cache.k_scale.cpu().double(), ks) and torch.equal(cache.v_scale.cpu().double(), vs)
        same_cells(cache.k, kc, False)
        same_cells(cache.v, vc, True)
    kd, vd = cache.read_pages(table[-1:, 0].to(dev).long())
    assert torch.equal(kd.cpu().double()[0], kc[table[-1, 0]] * ks[table[-1, 0]][:, None, None])
    assert torch.equal(vd.cpu().double()[0], vc[table[-1, 0]] * vs[table[-1, 0]][:, None, None])


def test_append_draft_then_rollback(hip_device):
    """A few tokens written, some taken back by a shorter length, others written in their place: scales stay, cells
    past the end keep their bytes until they are written again."""
    g = torch.Generator().manual_seed(12)
    dev, page, d, kv = hip_device, 32, 64, 1
    cache, (kc, ks, vc, vs) = filled(g, 4, kv, page, d, d, dev)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32)
    for lens, new, size in (([30, 20], [30, 20], 1.0), ([35, 24], [5, 4], 3.0), ([33, 21], [2, 1], 0.1), ([37, 33], [4, 12], 9.0)):
        n = sum(new)
        k, v = (size * torch.randn(n, kv, d, generator=g)).to(BF16), (size * torch.randn(n, kv, d, generator=g)).to(BF16)
        lengths, starts = torch.tensor(lens, dtype=torch.int32), torch.tensor([0, new[0], n], dtype=torch.int32)
        cache.append(k.to(dev), v.to(dev), table.to(dev), lengths.to(dev), starts.to(dev))
        for rows, c, s in ((k, kc, ks), (v, vc, vs)):
            R.append(c, s, rows, table, lengths, starts)
        assert torch.equal(cache.k_scale.cpu().double(), ks) and torch.equal(cache.v_scale.cpu().double(), vs)
        same_cells(cache.k, kc, False)
        same_cells(cache.v, vc, True)


def test_append_odd_batches(hip_device):
    """Non-finite values, zeros, tiny and huge ones; pages that are not there; more new tokens than positions; positions
    past the table; rows of no sequence; 64-bit lists; strided rows."""
    g = torch.Generator().manual_seed(11)
    page, d, kv, dev = 32, 64, 2, hip_device
    cache, (kc, ks, vc, vs) = filled(g, 12, kv, page, d, d, dev)
    table = torch.tensor([[3, 99], [-5, 4], [5, 6], [7, 8], [9, 10]])
    lengths = torch.tensor([40, 60, 20, 70, 9])
    starts = torch.tensor([2, 22, 52, 82, 122, 131])  # rows 0, 1 and from 131 on belong to nobody; the third has more than its 20
    n = 135
    k, v = torch.randn(n, kv, d, generator=g), torch.randn(n, kv, d, generator=g)
    k[10, 0, 3], k[11, 1, 0], k[12, 0, 5] = math.inf, math.nan, -math.inf
    k[122:131] = 0
    v[122:131] = 1e-33
    v[90] = 3e38
    wide = torch.zeros(n, kv, 2 * d)
    wide[..., :d] = v
    cache.append(k.to(dev), wide.to(dev)[..., :d], table.to(dev), lengths.to(dev), starts.to(dev))
    for rows, c, s in ((k, kc, ks), (v, vc, vs)):
        R.append(c, s, rows, table, lengths, starts)
    assert torch.equal(cache.k_scale.cpu().double(), ks) and torch.equal(cache.v_scale.cpu().double(), vs)
    same_cells(cache.k, kc, False)
    same_cells(cache.v, vc, True)
    # nothing at all
    before = cache.k.view(torch.uint8).clone()
    cache.append(k[:0].to(dev), v[:0].to(dev), table.to(dev)[:0], lengths.to(dev)[:0])
    cache.append(k[:0].to(dev), v[:0].to(dev), table.to(dev), lengths.to(dev), torch.zeros(6, dtype=torch.int32, device=dev))
    cache.append(k[:5].to(dev), v[:5].to(dev), table.to(dev)[:, :0], lengths.to(dev))
    assert torch.equal(cache.k.view(torch.uint8), before)


# ------------------------------------------------------------------ attention
def attend_close(y, lse, want, wlse, weight, size, p_top, dt, d, n_keys, sv):
    """A score is a sum of d exact products: 2 d 2^-24 of the sum of their sizes at most; x in units of log2 is
    rounded twice (2^-23 of its size each), exp2 by 2^-22: delta, relative, on each probability and on their sum,
    which has n 2^-24 of its own.  A probability is rounded to dt: half a step, and under f16's 2^-14 2^-25 of 64 at most.
    Then y is rounded once."""
    delta = (2 * d * 2.0 ** -24 + 3 * 2.0 ** -23) * size + 2.0 ** -21 + n_keys * 2.0 ** -24
    u = half_step(dt)
    tol = (u + 2 * delta)[:, None] * weight if torch.is_tensor(delta) else (u + 2 * delta) * weight
    if dt == F16:
        tol = tol + n_keys * 2.0 ** -25 * 448 * (p_top * sv)[:, None] + 2.0 ** -24
    tol = tol * (1 + u) + u * want.abs()
    assert bool(((y.cpu().double() - want).abs() <= tol + 1e-30).all()), float(((y.cpu().double() - want).abs() - tol).max())
    if lse is not None:
        fin = torch.isfinite(wlse)
        assert torch.equal(torch.isfinite(lse.cpu()), fin) and torch.equal(lse.cpu()[~fin].double(), wlse[~fin])
        assert bool(((lse.cpu().double() - wlse).abs() <= 2 * delta + 2.0 ** -22 * wlse.abs())[fin].all())


def check_attend(cache, plain, q, table, lengths, starts, y, lse, scale, causal, rows=None):
    kc, ks, vc, vs = plain
    k, v = kc * ks[:, :, None, None], vc * vs[:, :, None, None]
    for b in range(len(lengths)):
        first, end = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        n = int(lengths[b])
        kk, vv = R.sequence(k, table, b, n), R.sequence(v, table, b, n)
        for t in range(first, end):
            if rows is not None and t not in rows:
                continue
            seen = torch.arange(n) <= (n - (end - first) + t - first) if causal else torch.ones(n, dtype=torch.bool)
            want, wl, weight, size, p = R.attend(q[t].double(), kk, vv, seen, scale)
            top = p.amax(0) if p.shape[0] else q.new_zeros(q.shape[1]).double()
            attend_close(y[t], None if lse is None else lse[t], want, wl, weight, size, top, q.dtype, q.shape[2], n,
                         float(vs.max()))


@pytest.mark.parametrize("page,h,kv,d,dv,lens,new,causal,dt", [
    (64, 32, 4, 128, 128, [1, 64, 65, 777, 31, 32, 33], None, True, BF16),
    (32, 16, 2, 64, 64, [1, 5, 0, 300, 1500], None, True, F16),
    (64, 16, 16, 192, 128, [200, 129], None, True, F16),
    (128, 12, 4, 128, 128, [40, 300, 129], [40, 77, 0], True, BF16),   # groups of 3
    (64, 8, 1, 256, 256, [65, 200], [3, 4], True, BF16),
    (64, 9, 3, 192, 192, [70, 128], [70, 33], False, F16),
    (32, 40, 1, 64, 64, [95], [7], True, BF16),                         # 40 heads on one: two row tiles per token
    (64, 64, 1, 128, 128, [130, 3], None, True, F16),
    (64, 4, 4, 128, 128, [260, 100], [260, 50], True, F16),
    (32, 6, 1, 128, 128, [120, 64], [120, 64], True, BF16),
])
def test_attend(hip_device, page, h, kv, d, dv, lens, new, causal, dt):
    g = torch.Generator().manual_seed(page + h + d + len(lens))
    n = len(lens) if new is None else sum(new)
    counts = [-(-x // page) for x in lens]
    dev = hip_device
    cache, plain = filled(g, sum(counts) + 2, kv, page, d, dv, dev)
    table = table_of(g, counts, max(counts) + 1, sum(counts) + 2)
    starts = None if new is None else torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    q = (1.5 * torch.randn(n, h, d, generator=g)).to(dt)
    lengths = torch.tensor(lens, dtype=torch.int32)
    args = (table.to(dev), lengths.to(dev), None if starts is None else starts.to(dev))
    y, lse = cache.attend(q.to(dev), *args, causal=causal, return_lse=True)
    assert y.dtype == dt and y.shape == (n, h, dv) and lse.shape == (n, h)
    rows = None if n <= 130 else set(range(0, n, 7)) | {n - 1}
    check_attend(cache, plain, q, table, lengths, starts, y, lse, d ** -0.5, causal, rows)
    assert torch.equal(cache.attend(q.to(dev), *args, causal=causal), y)  # the same bits again


@pytest.mark.parametrize("n,page,dt", [(20000, 64, BF16), (33333, 32, F16)])
def test_attend_long(hip_device, n, page, dt):
    """Keys split over workgroups and joined; with a table much wider than what is used."""
    g = torch.Generator().manual_seed(n)
    dev = hip_device
    counts = [-(-n // page), 3]
    cache, plain = filled(g, sum(counts), 2, page, 64, 64, dev)
    table = table_of(g, counts, 2 * counts[0], sum(counts))
    lengths = torch.tensor([n, 2 * page + 1], dtype=torch.int32)
    q = (2 * torch.randn(2, 16, 64, generator=g)).to(dt)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), return_lse=True, scale=0.2)
    check_attend(cache, plain, q, table, lengths, None, y, lse, 0.2, True)
    imp = cache.importance(q.to(dev), table.to(dev), lengths.to(dev), scale=0.2)
    imp2 = cache.importance(q.to(dev), table.to(dev), lengths.to(dev), scale=0.2, lse=lse, out_len=n)
    check_importance(plain, q, table, lengths, 0.2, imp)
    check_importance(plain, q, table, lengths, 0.2, imp2)


@pytest.mark.parametrize("d,dv,dt,causal", [(64, 64, BF16, True), (128, 128, F16, True), (192, 128, BF16, False)])
def test_attend_many_rows(hip_device, d, dv, dt, causal):
    """Enough rows that a wave takes 64 of them (tokens times heads from 131072 on): two prompts with 256 heads to a key
    head, rows that end inside a tile, NaN among what later tokens bring."""
    g = torch.Generator().manual_seed(d + dv)
    dev, page, kv, h = hip_device, 32, 2, 512
    lens, new = [150, 133], [150, 110]
    counts = [5, 5]
    cache, plain = filled(g, 12, kv, page, d, dv, dev)
    table = table_of(g, counts, 6, 12)
    if causal:  # position 141 of the first prompt, in V: later tokens see it
        plain[2][table[0, 4], 1, 13, 7] = math.nan
        cache.v.view(torch.uint8).copy_(R.pack(plain[2], True).view(torch.uint8))
    lengths, starts = torch.tensor(lens, dtype=torch.int32), torch.tensor([0, 150, 260], dtype=torch.int32)
    q = (1.5 * torch.randn(260, h, d, generator=g)).to(dt)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev), causal=causal, return_lse=True)
    if causal:
        bad = torch.isnan(y).cpu()
        assert bool(bad[141:150, 256:, 7].all()) and int(bad.sum()) == 9 * 256
        y = torch.where(torch.isnan(y), torch.zeros_like(y), y)
        plain[2] = torch.nan_to_num(plain[2])
    rows = {0, 1, 31, 64, 127, 140, 150, 151, 200, 259} if causal else {0, 149, 150, 222}
    check_attend(cache, plain, q, table, lengths, starts, y, lse, d ** -0.5, causal, rows)


def test_attend_small_scales(hip_device):
    """Values so small that their scales sit at the floor of 2^-100."""
    g = torch.Generator().manual_seed(77)
    dev, d = hip_device, 64
    from table_moe.ops import Fp8KVCache

    cache = Fp8KVCache(20, 1, d, page_size=32, device=dev)
    k, v = torch.randn(600, 1, d, generator=g), torch.randn(600, 1, d, generator=g) * 1e-29
    table, lengths = torch.arange(20, dtype=torch.int32, device=dev)[None], torch.tensor([600], device=dev)
    cache.append(k.to(dev), v.to(dev), table, lengths, torch.tensor([0, 600], device=dev))
    assert float(cache.v_scale[:19].max()) == 2.0 ** -100
    q = torch.randn(1, 4, d, generator=g).to(BF16)
    y, lse = cache.attend(q.to(dev), table, lengths, return_lse=True)
    kk, vv = (t.cpu().double().transpose(1, 2).flatten(0, 1)[:600] for t in cache.read_pages())
    # (bf16 holds these magnitudes: its exponents are fp32's)
    want = R.attend(q[0].double(), kk, vv, torch.ones(600, dtype=torch.bool), d ** -0.5)
    attend_close(y[0].float() * 2.0 ** 90, lse[0], want[0] * 2.0 ** 90, want[1], want[2] * 2.0 ** 90, want[3], want[4].amax(0), BF16,
                 d, 600, 1.0)


def test_attend_offsets_past_32_bits(hip_device):
    """Pages whose bytes lie past 2^32, and rows whose elements do not start at 0."""
    dev = hip_device
    from table_moe.ops import Fp8KVCache

    page, d, kv = 128, 256, 4  # 128 KiB a page for K, as much for V
    cache = Fp8KVCache(36000, kv, d, d, page, device=dev)  # 4.7e9 bytes each
    g = torch.Generator().manual_seed(3)
    table = torch.tensor([[35999, 17, 33000]], dtype=torch.int32)
    lengths = torch.tensor([300], dtype=torch.int32)
    starts = torch.tensor([0, 300], dtype=torch.int32)
    k, v = torch.randn(300, kv, d, generator=g).to(BF16), torch.randn(300, kv, d, generator=g).to(BF16)
    cache.append(k.to(dev), v.to(dev), table.to(dev), lengths.to(dev), starts.to(dev))
    small = [table[0].long().to(dev)]
    kc, vc = (R.raw(t.view(torch.uint8)[small[0]].view(t.dtype), i == 1) for i, t in enumerate((cache.k, cache.v)))
    ks, vs = cache.k_scale[small[0]].cpu().double(), cache.v_scale[small[0]].cpu().double()
    wk, wv = torch.zeros_like(kc), torch.zeros_like(vc)
    ws, wt = torch.ones_like(ks), torch.ones_like(vs)
    local = torch.tensor([[0, 1, 2]])
    R.append(wk, ws, k, local, lengths, starts)
    R.append(wv, wt, v, local, lengths, starts)
    assert torch.equal(kc, wk) and torch.equal(vc, wv) and torch.equal(ks, ws) and torch.equal(vs, wt)
    q = torch.randn(300, 8, d, generator=g).to(BF16)
    y = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev))
    check_attend(cache, (kc, ks, vc, vs), q, local, lengths, starts, y, None, d ** -0.5, True, {0, 1, 127, 128, 299})


def test_attend_what_is_not_seen(hip_device):
    """NaN and leftovers past a sequence's end, NaN that later tokens bring, pages that are not there, rows that see
    nothing, rows of no sequence."""
    g = torch.Generator().manual_seed(8)
    dev, page, d, kv, h = hip_device, 64, 128, 2, 8
    cache, plain = filled(g, 6, kv, page, d, d, dev)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    lengths, starts = torch.tensor([70, 100], dtype=torch.int32), torch.tensor([0, 70, 170], dtype=torch.int32)
    token, col = R.cells(page, d, False)
    for c, packed, values in ((plain[0], cache.k, False), (plain[2], cache.v, True)):
        c[1, :, 6:] = math.nan   # past the first's end
        c[3, :, 36:] = math.nan
        c[3, 1, 10] = math.nan   # position 74 of the second: later tokens see it, earlier ones do not
        packed.view(torch.uint8).copy_(R.pack(c, values).view(torch.uint8))
    q = torch.randn(172, h, d, generator=g).to(BF16)
    out = torch.full((172, h, d), 7.0, dtype=BF16, device=dev)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev), out=out, return_lse=True)
    assert y is out and bool((out[170:] == 7).all())
    finite = torch.isfinite(y[:170]).all(-1).cpu()
    assert bool(finite[:144].all()) and bool(finite[144:, :4].all()) and not bool(finite[144:, 4:].any())
    clean = [torch.nan_to_num(t) for t in plain]
    check_attend(cache, clean, q, table, lengths, starts, y, lse, d ** -0.5, True, {0, 5, 6, 7, 69, 70, 100, 143})
    # V's NaN alone, in one column: that column of the rows that see it
    cache2, plain2 = filled(g, 2, 1, page, d, d, dev)
    plain2[2][0, 0, 40, 77] = math.nan
    cache2.v.view(torch.uint8).copy_(R.pack(plain2[2], True).view(torch.uint8))
    q2 = torch.randn(64, 1, d, generator=g).to(F16)
    y2 = cache2.attend(q2.to(dev), torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([64], device=dev),
                       torch.tensor([0, 64], device=dev))
    bad = torch.isnan(y2[:, 0]).cpu()
    assert int(bad.sum()) == 24 and bool(bad[40:, 77].all())
    # a page that is not there: as if the rest were all; no page at all; no token
    t3 = torch.tensor([[0, 9], [-1, 2], [6, -7]], dtype=torch.int32)
    l3 = torch.tensor([100, 120, 50], dtype=torch.int32)
    y3, lse3 = cache.attend(q[:3].to(dev), t3.to(dev), l3.to(dev), return_lse=True)
    kk, vv = clean[0] * clean[1][:, :, None, None], clean[2] * clean[3][:, :, None, None]
    for b, (p, n) in enumerate(((0, 64), (2, 56))):
        want = R.attend(q[b].double(), kk[p].transpose(0, 1)[:n], vv[p].transpose(0, 1)[:n], torch.ones(n, dtype=torch.bool), d ** -0.5)
        attend_close(y3[b], lse3[b], *want[:4], want[4].amax(0), BF16, d, n, float(clean[3].max()))
    assert bool((y3[2] == 0).all()) and bool((lse3[2] == -math.inf).all())
    i3 = cache.importance(q[:3].to(dev), t3.to(dev), l3.to(dev))
    assert bool((i3[0, 64:] == 0).all()) and bool((i3[1, :64] == 0).all()) and bool((i3[2] == 0).all())
    assert torch.allclose(i3.sum(1)[:2], torch.ones(2, device=dev), atol=1e-5)
    # more new tokens than positions: the first see nothing
    y4, lse4 = cache.attend(q[:10].to(dev), table[:1].to(dev), torch.tensor([4], device=dev), torch.tensor([0, 10], device=dev),
                            return_lse=True)
    assert bool((y4[:6] == 0).all()) and bool((lse4[:6] == -math.inf).all()) and bool(torch.isfinite(lse4[6:]).all())
    # a length past the table ends with it
    y5 = cache.attend(q[:1].to(dev), table[:1, :1].to(dev), torch.tensor([1 << 30], device=dev))
    want = R.attend(q[0].double(), kk[0].transpose(0, 1), vv[0].transpose(0, 1), torch.ones(64, dtype=torch.bool), d ** -0.5)
    attend_close(y5[0], None, *want[:4], want[4].amax(0), BF16, d, 64, float(clean[3].max()))
    # a negative length, starts that go back or past the rows: nothing faults
    cache.attend(q.to(dev), table.to(dev), torch.tensor([-3, 5], device=dev), torch.tensor([50, -4, 1 << 30], device=dev))
    cache.attend(q[:2].to(dev), table[:, :0].to(dev), lengths.to(dev))
    assert cache.attend(q[:0].to(dev), table[:0].to(dev), lengths[:0].to(dev)).shape == (0, h, d)


def test_attend_scales_far_apart_and_large_scores(hip_device):
    """Pages whose scales differ by 2^40, scores in the hundreds, a growing maximum over the tiles."""
    g = torch.Generator().manual_seed(21)
    dev, page, d, kv = hip_device, 32, 64, 1
    cache, plain = filled(g, 8, kv, page, d, d, dev)
    for p in range(8):
        plain[3][p] *= 2.0 ** (10 * (p % 4) - 20)
        plain[0][p] *= 2.0 ** -3
        plain[1][p] *= 2.0 ** (p - 1)
    cache.k.view(torch.uint8).copy_(R.pack(R.e4m3(plain[0]), False).view(torch.uint8))
    plain[0] = R.raw(cache.k, False)
    cache.k_scale.copy_(plain[1].float())
    cache.v_scale.copy_(plain[3].float())
    table = torch.arange(8, dtype=torch.int32)[None]
    q = (8 * torch.randn(250, 2, d, generator=g)).to(BF16)
    lengths, starts = torch.tensor([250], dtype=torch.int32), torch.tensor([0, 250], dtype=torch.int32)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev), return_lse=True)
    check_attend(cache, plain, q, table, lengths, starts, y, lse, d ** -0.5, True, set(range(0, 250, 11)) | {249})


@pytest.mark.parametrize("order,one_token", [("big first", False), ("big last", False), ("by turns", False), ("big first", True),
                                             ("big last", True), ("all big", True)])
def test_attend_value_scales_of_any_ratio(hip_device, order, one_token):
    """Value scales from 2^-100 to 2^120 among keys of like probability: each counts in the sum. One token of 2048 keys
    has its keys split over workgroups; pages of 32 go to the four waves in turn."""
    g = torch.Generator().manual_seed(31)
    dev, page, d, kv, pages = hip_device, 32, 64, 1, 64 if one_token else 16
    cache, plain = filled(g, pages, kv, page, d, d, dev)
    big = {"big first": lambda p: p < pages // 2, "big last": lambda p: p >= pages // 2, "by turns": lambda p: p % 2 == 0,
           "all big": lambda p: True}[order]
    for p in range(pages):
        plain[3][p] = 2.0 ** (120 if big(p) else -100)
    plain[2] *= 1 / 4.0  # (means of them stay under bf16's largest)
    cache.v.view(torch.uint8).copy_(R.pack(R.e4m3(plain[2]), True).view(torch.uint8))
    plain[2] = R.raw(cache.v, True)
    cache.v_scale.copy_(plain[3].float())
    table, n = torch.arange(pages, dtype=torch.int32)[None], pages * page
    t = 1 if one_token else n
    q = (0.5 * torch.randn(t, 4, d, generator=g)).to(BF16)
    lengths, starts = torch.tensor([n], dtype=torch.int32), None if one_token else torch.tensor([0, n], dtype=torch.int32)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), None if one_token else starts.to(dev), return_lse=True)
    # (in units of 2^120, where the tolerance's own arithmetic holds them)
    plain[3] = plain[3] * 2.0 ** -120
    check_attend(cache, plain, q, table, lengths, starts, y.double() * 2.0 ** -120, lse, d ** -0.5, True,
                 None if one_token else set(range(0, n, 37)) | {n - 1})


@pytest.mark.parametrize("h,kv,seqs,longest", [(4, 2, 64, 21000), (16, 8, 66, 20000), (40, 1, 70, 41000)])
def test_attend_lengths_that_differ(hip_device, h, kv, seqs, longest):
    """One long sequence among many short ones, one token each: its keys are split, theirs are not."""
    g = torch.Generator().manual_seed(seqs)
    dev, page, d = hip_device, 128, 64
    lens = [int(x) for x in torch.randint(0, 700, (seqs,), generator=g)]
    lens[seqs // 2], lens[3], lens[4], lens[5] = longest, 0, 1, 4200
    counts = [-(-x // page) for x in lens]
    cache, plain = filled(g, sum(counts) + 1, kv, page, d, d, dev)
    table, lengths = table_of(g, counts, max(counts), sum(counts) + 1), torch.tensor(lens, dtype=torch.int32)
    q = (1.5 * torch.randn(seqs, h, d, generator=g)).to(BF16)
    args = (q.to(dev), table.to(dev), lengths.to(dev))
    y, lse = cache.attend(*args, return_lse=True)
    imp = cache.importance(*args)
    some = [0, 3, 4, 5, seqs // 2, seqs - 1]
    check_attend(cache, plain, q, table, lengths, None, y, lse, d ** -0.5, True, set(some))
    check_importance(plain, q[some], table[some], lengths[some], d ** -0.5, imp[some])
    # the others alone, whose table is narrow: the same up to two roundings of the result and those of its sums
    rest = [i for i in range(seqs) if i not in (seqs // 2, 5)]
    z = cache.attend(q[rest].to(dev), table[rest, :6].contiguous().to(dev), lengths[rest].to(dev))
    assert bool(((z.double() - y[rest].double()).abs() <= 2 * half_step(BF16) * y[rest].double().abs() + 1e-5 * 448 * float(plain[3].max())).all())


@pytest.mark.parametrize("h,kv,lens,new,page", [
    (8, 2, [5000, 0, 3000, 40], [3, 0, 2, 1], 64), (12, 4, [6000], [33], 32), (40, 1, [4100, 2000], [2, 2], 128),
    (4, 4, [2000] * 9, [4] * 9, 64), (8, 8, [300] * 40, [2] * 40, 64)])
def test_attend_drafted_tokens(hip_device, h, kv, lens, new, page):
    """A few new tokens for each of some sequences, keys split; rows behind the last sequence are left as they were."""
    g = torch.Generator().manual_seed(len(lens) + h)
    dev, d = hip_device, 128
    counts = [-(-x // page) for x in lens]
    cache, plain = filled(g, sum(counts) + 1, kv, page, d, d, dev)
    table, lengths = table_of(g, counts, max(counts), sum(counts) + 1), torch.tensor(lens, dtype=torch.int32)
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    n = sum(new)
    q = (1.5 * torch.randn(n + 3, h, d, generator=g)).to(BF16)
    out = torch.full((n + 3, h, d), 7.0, dtype=BF16, device=dev)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev), out=out, return_lse=True)
    assert bool((y[n:] == 7).all())
    check_attend(cache, plain, q, table, lengths, starts, y, lse, d ** -0.5, True, set(range(0, n, 5)) | {n - 1})


@pytest.mark.parametrize("h,kv,d,dv,lens,new", [
    (8, 2, 64, 64, [17000, 30, 9000, 17000, 1100], [1, 1, 4, 2, 1100]),     # the prompt's rows fill the device
    (8, 2, 192, 128, [17000, 700, 4500], [3, 300, 0]),                      # all are split
    (64, 8, 64, 64, [33000, 2100, 5, 33000], [1, 2100, 5, 3]),              # 64 rows a wave
])
def test_attend_long_sequences_beside_a_prompt(hip_device, h, kv, d, dv, lens, new):
    """Single and drafted tokens of long sequences in one call with a prompt: their keys are split, the prompt's may not be."""
    g = torch.Generator().manual_seed(sum(lens))
    dev, page = hip_device, 128
    counts = [-(-x // page) for x in lens]
    cache, plain = filled(g, sum(counts) + 1, kv, page, d, dv, dev)
    table, lengths = table_of(g, counts, max(counts), sum(counts) + 1), torch.tensor(lens, dtype=torch.int32)
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    n = sum(new)
    q = (1.5 * torch.randn(n, h, d, generator=g)).to(BF16)
    y, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev), return_lse=True)
    some = {0, 1, 2, 7, n // 2, n - 4, n - 2, n - 1}
    check_attend(cache, plain, q, table, lengths, starts, y, lse, d ** -0.5, True, some)


# ----------------------------------------------------------------- importance
def check_importance(plain, q, table, lengths, scale, got):
    k = plain[0] * plain[1][:, :, None, None]
    d = q.shape[2]
    for b in range(len(lengths)):
        n = int(lengths[b])
        kk = R.sequence(k, table, b, n)
        _, _, _, size, p = R.attend(q[b].double(), kk, kk, torch.ones(n, dtype=torch.bool), scale)
        want, m = p.mean(1), min(n, got.shape[1])
        # as in attend_close, the score's error twice (its own and the sum's)
        delta = float(size.max()) * (2 * d * 2.0 ** -24 + 3 * 2.0 ** -23) + 2.0 ** -21 + n * 2.0 ** -24
        assert bool(((got[b, :m].cpu().double() - want[:m]).abs() <= 4 * delta * want[:m] + 1e-37).all())
        assert bool((got[b, m:] == 0).all())


@pytest.mark.parametrize("page,h,kv,d,lens,dt", [
    (64, 32, 4, 128, [777, 1, 64], BF16), (32, 16, 16, 192, [100, 33], F16), (128, 12, 2, 64, [500], BF16),
    (64, 40, 1, 64, [90, 0], F16), (64, 24, 8, 192, [65], BF16), (64, 8, 1, 256, [300, 31], F16), (32, 3, 3, 128, [200], BF16)])
def test_importance(hip_device, page, h, kv, d, lens, dt):
    from table_moe.utils import ModalityContext
    from table_moe.utils.importance import cached_importance

    g = torch.Generator().manual_seed(h + d + lens[0])
    counts = [-(-x // page) for x in lens]
    dev = hip_device
    dv = 128 if d == 192 and page == 32 else d
    cache, plain = filled(g, sum(counts) + 1, kv, page, d, dv, dev)
    table, lengths = table_of(g, counts, max(counts), sum(counts) + 1), torch.tensor(lens, dtype=torch.int32)
    q = (1.5 * torch.randn(len(lens), h, d, generator=g)).to(dt)
    args = (q.to(dev), table.to(dev), lengths.to(dev))
    got = cache.importance(*args)
    assert got.shape == (len(lens), max(counts) * page)
    check_importance(plain, q, table, lengths, d ** -0.5, got)
    _, lse = cache.attend(*args, return_lse=True)
    again = cached_importance(cache, *args, lse=lse, query_length=max(lens) - 5 if max(lens) > 5 else 1)
    check_importance(plain, q, table, lengths, d ** -0.5, again)
    assert torch.equal(ModalityContext.get_attn_weights(), again.reshape(-1))
    assert cached_importance(cache, q.to(dev).float(), *args[1:]) is None and ModalityContext.get_attn_weights() is None
    assert cache.importance(*args, out_len=0).shape == (len(lens), 0)
    long = cache.importance(*args, out_len=max(counts) * page + 77)
    assert torch.equal(long[:, :got.shape[1]], got) and bool((long[:, got.shape[1]:] == 0).all())


# ------------------------------------------------------------------- together
def test_together_captured(hip_device):
    """Rotate, append, attend and importance as a layer runs them, prompt and decode steps, eager and captured; the
    importance chooses experts.  Replays with other inputs in the same buffers equal eager runs."""
    from table_moe.ops import Fp8KVCache, rotate_positions
    from table_moe.skip.pruning import build_prefill_keep_mask

    dev = hip_device
    g = torch.Generator().manual_seed(31)
    h, kv, d, page, b = 8, 2, 128, 64, 3
    inv = (1e6 ** (-torch.arange(64).double() / 64)).float().to(dev)
    lens = [70, 128, 9]
    table = torch.arange(b * 4, dtype=torch.int32, device=dev).view(b, 4).flip(1).contiguous()
    starts = torch.tensor([0, 70, 198, 207], dtype=torch.int32, device=dev)
    mk = lambda n, heads: torch.randn(n, heads, d, generator=g).to(BF16).to(dev)  # noqa: E731

    def layer(cache, q, k, v, pos, lengths, starts):
        q, k = rotate_positions(q, k, pos, inv, (24, 20, 20), interleaved=True)
        cache.append(k, v, table, lengths, starts)
        y, lse = cache.attend(q, table, lengths, starts, return_lse=True)
        last = torch.arange(b, device=dev) if starts is None else starts[1:].long() - 1
        return y, cache.importance(q[last], table, lengths, lse=lse[last]), cache.importance(q[last], table, lengths)

    def prompt(cache):
        return layer(cache, *data, pos, lengths, starts)

    data = (mk(207, h), mk(207, kv), mk(207, kv))
    pos = torch.randint(0, 200, (3, 207), generator=g).to(dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    eager = Fp8KVCache(12, kv, d, page_size=page, device=dev)
    y, imp, imp2 = prompt(eager)
    assert torch.allclose(imp, imp2, rtol=1e-4) and torch.allclose(imp.sum(1), torch.ones(b, device=dev), atol=1e-4)
    sel = torch.stack([torch.randperm(16, generator=g)[:4] for _ in range(70)]).to(dev)
    keep = build_prefill_keep_mask(sel, torch.full((70, 4), 0.25, device=dev), imp[0, :70].contiguous(), 16, 0.5)
    assert 0 < int(keep.sum()) < keep.numel()

    captured = Fp8KVCache(12, kv, d, page_size=page, device=dev)
    assert all(torch.equal(a, c) for a, c in zip(prompt(captured), (y, imp, imp2)))
    # decode steps: buffers that the graph reads
    q1, k1, v1, pos1 = mk(b, h), mk(b, kv), mk(b, kv), torch.zeros(3, b, dtype=torch.long, device=dev)
    len1 = lengths.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    scratch = Fp8KVCache.wrap(captured.k.clone(), captured.v.clone(), captured.k_scale.clone(), captured.v_scale.clone())
    with torch.cuda.stream(side):
        layer(scratch, q1, k1, v1, pos1, len1, None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg, ig, ig2 = layer(captured, q1, k1, v1, pos1, len1, None)
    for step in range(6):
        q1.copy_(mk(b, h)), k1.copy_(mk(b, kv) * (1 + step)), v1.copy_(mk(b, kv))
        len1.add_(1)
        pos1.copy_((len1 - 1).long().expand(3, b))
        graph.replay()
        torch.cuda.synchronize()
        ye, ie, ie2 = layer(eager, q1, k1, v1, pos1, len1, None)
        torch.cuda.synchronize()
        assert torch.equal(yg, ye) and torch.equal(ig, ie) and torch.equal(ig2, ie2), step
        assert torch.equal(captured.k.view(torch.uint8), eager.k.view(torch.uint8)) and torch.equal(captured.v_scale, eager.v_scale)


def test_two_calls_at_once(hip_device):
    """Calls on two streams share nothing."""
    g = torch.Generator().manual_seed(9)
    dev = hip_device
    cache, plain = filled(g, 40, 2, 64, 128, 128, dev)
    table = torch.randperm(40, generator=g).to(torch.int32).view(1, 40).to(dev)
    lengths = torch.tensor([2500], dtype=torch.int32, device=dev)
    qs = [torch.randn(1, 16, 128, generator=g).to(BF16).to(dev) for _ in range(2)]
    want = [cache.attend(q, table, lengths) for q in qs]
    wi = [cache.importance(q, table, lengths) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((cache.attend(qs[i], table, lengths), cache.importance(qs[i], table, lengths)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) and torch.equal(p, wi[i]) for y, p in got[i])


def test_cache_refusals(hip_device):
    from table_moe.ops import Fp8KVCache

    dev = hip_device
    for kw in (dict(page_size=48), dict(head_dim=96), dict(v_dim=64), dict(n_pages=0), dict(n_kv_heads=0)):
        with pytest.raises(ValueError):
            Fp8KVCache(**{**dict(n_pages=2, n_kv_heads=2, head_dim=128, device=dev), **kw})
    with pytest.raises(RuntimeError):
        Fp8KVCache(2, 2, 128, device="cpu")
    c = Fp8KVCache(4, 2, 128, device=dev)
    ok = [c.k, c.v, c.k_scale, c.v_scale]
    Fp8KVCache.wrap(*ok)
    for i, t in ((0, c.k.view(torch.uint8)), (0, c.k[:2]), (0, c.k.transpose(0, 1)), (1, c.v[..., :8]), (2, c.k_scale.half()),
                 (3, c.v_scale[:2]), (0, c.k[:, :, :, :2])):
        with pytest.raises(ValueError):
            Fp8KVCache.wrap(*[t if j == i else o for j, o in enumerate(ok)])
    q, kv = torch.zeros(3, 4, 128, dtype=BF16, device=dev), torch.zeros(3, 2, 128, dtype=BF16, device=dev)
    t, n = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    bad_rows = dict(table=[t[:2], t[0], t.float()], lengths=[n[:2], t, n.float()], starts=[n, n.float()])
    for name, values in bad_rows.items():
        for x in values:
            kw = {**dict(table=t, lengths=n, starts=None), name: x}
            with pytest.raises(ValueError):
                c.append(kv, kv, **kw)
            with pytest.raises(ValueError):
                c.attend(q, **kw)
            if name != "starts":
                with pytest.raises(ValueError):
                    c.importance(q, **{k: v for k, v in kw.items() if k != "starts"})
    with pytest.raises(ValueError, match="overlap"):
        c.attend(q, t, n, out=q)
    for k, v in ((kv[:, :1], kv), (kv, kv.half()), (kv.double(), kv.double()), (kv[..., :64], kv), (kv[:2], kv)):
        with pytest.raises(ValueError):
            c.append(k, v, t, n)
    for x in (q.float(), q[:, :3], q[..., :64], q[:, :0], q[:2]):
        with pytest.raises(ValueError):
            c.attend(x, t, n)
        with pytest.raises(ValueError):
            c.importance(x, t, n)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(out=q[:, :2]),
               dict(out=torch.zeros(3, 4, 128, device=dev)), dict(out=q[:1].expand(3, 4, 128)),
               dict(out=torch.zeros(3 * 4 * 128 + 4, dtype=BF16, device=dev)[4:].view(3, 4, 128))):
        with pytest.raises(ValueError):
            c.attend(q, t, n, **kw)
    for kw in (dict(scale=0.0), dict(lse=torch.zeros(3, 3, device=dev)), dict(lse=torch.zeros(3, 4, device=dev, dtype=F16)),
               dict(out_len=-1)):
        with pytest.raises(ValueError):
            c.importance(q, t, n, **kw)
    with pytest.raises(RuntimeError):
        c.attend(q.cpu(), t, n)

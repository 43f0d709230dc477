"""Attention and importance over the 8-bit cache where keys are split over workgroups and joined: each tile and each
key counts once, at every width of columns, in decode steps, drafted tokens and calls of mixed lengths."""

import ctypes as C
import math

import pytest
import torch

from kv8_exact import LN2, Inputs, accepts, by_column, tolerances

BF16, F16 = torch.bfloat16, torch.float16
gpu = pytest.mark.gpu

SHORT = [int(x) for x in torch.randint(0, 700, (40,), generator=torch.Generator().manual_seed(2))]

# page, heads, key heads, columns of K and V, lengths, new tokens (None: one each), type, parts: "few" or "many", as the
# joining kernel has two forms, up to four times the sets of v_dim / 4 threads that 256 hold and above ("": either)
CASES = {
    "64 columns, 128 parts": (64, 16, 2, 64, 64, [20001], None, BF16, "many"),
    "64 columns, two sequences": (32, 16, 2, 64, 64, [33333, 65], None, F16, ""),
    "128 columns, 32 parts or less": (64, 16, 2, 128, 128, [4000], None, BF16, "few"),
    "128 columns, more": (64, 16, 1, 128, 128, [9000], None, F16, "many"),
    "192 to 128 columns": (32, 16, 4, 192, 128, [5001], None, BF16, "many"),
    "192 columns, 20 parts or less": (32, 6, 2, 192, 192, [2000], None, BF16, "few"),
    "192 columns, 20 parts or less, f16": (128, 24, 8, 192, 192, [2049], None, F16, "few"),
    "192 columns, more": (128, 24, 8, 192, 192, [9000], None, F16, "many"),
    "192 columns, more, bf16": (64, 3, 1, 192, 192, [3001], None, BF16, "many"),
    "256 columns, 16 parts or less": (64, 8, 1, 256, 256, [1500], None, F16, "few"),
    "256 columns, 16 parts or less, bf16": (32, 8, 4, 256, 256, [1999], None, BF16, "few"),
    "256 columns, more": (64, 8, 1, 256, 256, [5003], None, BF16, "many"),
    "256 columns, 128 parts": (128, 8, 1, 256, 256, [16500], None, F16, "many"),
    "40 heads on one": (64, 40, 1, 256, 256, [3000], None, BF16, "many"),
    "drafted, 192 columns": (64, 8, 2, 192, 192, [5000, 0, 3000, 40], [3, 0, 2, 1], BF16, ""),
    "drafted, 256 columns": (64, 8, 1, 256, 256, [4100, 2000], [2, 5], F16, ""),
    "drafted, 64 columns": (32, 12, 4, 64, 64, [6000], [33], F16, ""),
    "one long among short, 256 columns": (64, 4, 1, 256, 256, [17000, *SHORT], None, BF16, ""),
    "one long among short, 192 columns": (128, 24, 8, 192, 192, [*SHORT, 12000, 0, 1], None, F16, ""),
    "one long among many short, 64 columns": (128, 40, 1, 64, 64, [*SHORT, 41000, *SHORT], None, BF16, ""),
    "prompt beside long ones, 192 columns": (128, 8, 2, 192, 192, [17000, 700, 4500], [3, 300, 0], F16, ""),
    "prompt beside long ones, 256 columns": (64, 8, 1, 256, 256, [9000, 1100, 9000], [1, 1100, 2], BF16, ""),
    "64 rows a wave, split": (128, 64, 8, 64, 64, [33000, 2100, 33000], [1, 2100, 3], F16, ""),
}


def inputs(name):
    page, h, kv, d, dv, lens, new, dt, _ = CASES[name]
    return Inputs(len(name), page, h, kv, d, dv, lens, new, dt)


def some(inp):
    """Rows to check: all of a small call, else the first and last of each sequence and some between."""
    rows = list(inp.rows())
    if len(rows) <= 90:
        return rows
    ends = {sum(inp.new[:b]) + i for b, m in enumerate(inp.new) for i in (0, 1, m - 1) if 0 <= i < m}
    return [r for r in rows if r[0] in ends or r[0] % 173 == 5]


def splits_of(cache, inp, dev):
    from table_moe import _native as N

    batch, _ = cache._batch(*(inp.args(dev) + (None,))[:3], inp.q.shape[0])
    nbytes = N.lib().tm_kv8_attention_workspace_size(cache._ref, C.byref(batch), inp.h)
    return (nbytes - 16) // (inp.q.shape[0] * inp.h * (inp.dv + 2) * 4) if nbytes else 1


@pytest.mark.parametrize("name", CASES)
def test_the_tolerance_sees_a_tile(name):
    """A result without one of the tiles, or with one of them twice, is off by more than is allowed, whichever tile:
    some query head of every key head says so."""
    inp = inputs(name)
    longest = max(range(len(inp.lens)), key=lambda b: (inp.new[b] > 0) * inp.lens[b])
    row, b, seen = [r for r in inp.rows() if r[1] == longest][-1]
    w, wv = inp.tiles(row, b, seen)
    total, sums = w.sum(0), by_column(inp, b, wv)
    assert bool(accepts(sums / total[:, None], torch.log(total), sums, total, seen, inp.dt).all())
    cols = inp.column(b, 32 * torch.arange(len(w)))
    for sign in (-1, 1):
        for t in range(len(w)):
            other = sums.clone()
            other[:, cols[t]] += sign * wv[t]
            less = total + sign * w[t]
            got = (other / less[:, None]).to(inp.dt).double()
            ok = accepts(got, torch.log(less), sums, total, seen, inp.dt).view(inp.kv, -1).all(1)
            assert not bool(ok.any()), (t, sign)


@gpu
@pytest.mark.parametrize("name", CASES)
def test_each_tile_counts_once(hip_device, name):
    inp, dev, parts = inputs(name), hip_device, CASES[name][-1]
    cache = inp.cache(dev)
    if parts:
        n, most = splits_of(cache, inp, dev), 4 * (256 // (inp.dv // 4))
        assert 1 < n <= most if parts == "few" else n > most, n
    q = inp.q.to(inp.dt).to(dev)
    y, lse = cache.attend(q, *inp.args(dev), scale=LN2, return_lse=True)
    y, lse = y.cpu().double(), lse.cpu().double()
    for row, b, seen in some(inp):
        if seen == 0:
            assert bool((y[row] == 0).all()) and bool((lse[row] == -math.inf).all())
            continue
        w, wv = inp.tiles(row, b, seen)
        ok = accepts(y[row], lse[row], by_column(inp, b, wv), w.sum(0), seen, inp.dt)
        assert bool(ok.all()), (row, b, seen, (~ok).nonzero().flatten().tolist())


@gpu
@pytest.mark.parametrize("name", [n for n, c in CASES.items() if c[6] is None])
def test_each_key_counts_in_the_importance(hip_device, name):
    """Without a log sum exp: the statistics of split keys, at every head_dim."""
    inp, dev = inputs(name), hip_device
    cache = inp.cache(dev)
    got = cache.importance(inp.q.to(inp.dt).to(dev), *inp.args(dev), scale=LN2).cpu().double()
    for row, b, seen in inp.rows():
        if seen:
            p = inp.weights(row, b, seen)
            want = (p / p.sum(0)).mean(1)
            tol = 2 * tolerances(seen, inp.dt)[0] + inp.h * 2.0 ** -24
            assert bool(((got[b, :seen] - want).abs() <= tol * want).all()), (b, seen)
        assert bool((got[b, seen:] == 0).all())


@gpu
@pytest.mark.parametrize("page,h,kv,d,dv,n,new,dt", [
    (64, 64, 1, 64, 64, 9001, 1, BF16), (32, 64, 1, 128, 128, 4100, 2, F16), (64, 48, 1, 192, 192, 2100, 4, F16),
    (64, 48, 1, 192, 192, 6007, 4, BF16), (128, 64, 1, 256, 256, 1600, 4, BF16), (64, 64, 1, 256, 256, 5003, 4, F16),
])
def test_first_and_last_key_of_each_tile(hip_device, page, h, kv, d, dv, n, new, dt):
    """Each of these keys in turn has 2^20 times the weight of any other: the result is its value, and no key counts twice."""
    dev = hip_device
    inp = Inputs(n + d, page, h, kv, d, dv, [n], [new] if new > 1 else None, dt)
    g = torch.Generator().manual_seed(n)
    v = torch.randint(-7, 8, (n, kv, dv), generator=g).double()
    keys = torch.arange(0, n - new, 32)  # (what the first of the new tokens sees, too)
    targets = torch.cat([keys, (keys + 31).clamp(max=n - new)])
    rows = new * h
    assert rows >= d
    for part in targets.split(d):
        k = torch.zeros(n, kv, d, dtype=torch.float64)
        k[part, :, torch.arange(len(part))] = 20.0
        inp.ks.fill_(1.0)
        cache = inp.cache(dev, [k], [v])
        column = torch.arange(rows) % len(part)
        q = torch.zeros(rows, d, dtype=torch.float64)
        q[torch.arange(rows), column] = 1.0
        y, lse = cache.attend(q.view(new, h, d).to(dt).to(dev), *inp.args(dev), scale=LN2, return_lse=True)
        y, lse = y.cpu().double().view(rows, dv), lse.cpu().double().view(rows)
        seen = n - new + 1 + torch.arange(new).repeat_interleave(h)
        total = 2.0 ** 20 + seen - 1.0
        upto = v[:, 0].cumsum(0)
        chosen = v[part[column], 0]
        sums = upto[seen - 1] + (2.0 ** 20 - 1) * chosen
        # the error of what is small is counted on the sizes, 7 each
        delta, u = tolerances(n, dt)
        delta += 2 * math.log(2) * (3 * 12 + 2 * 24) * 2.0 ** -24  # (scores up to 20)
        want, size = sums / total[:, None], ((2.0 ** 20 - 1) * chosen.abs() + upto.new_tensor(7.0) * seen[:, None]) / total[:, None]
        # weights 2^-12 of the first reference are under fp16's normal numbers: 2^-25 each where the largest has 2^8 or more
        lost = seen[:, None] * 7 * 2.0 ** -33
        assert bool(((y - want).abs() <= 2 * delta * size + lost + u * (want.abs() + 2 * delta * size + lost)).all()), part[0]
        assert bool(((lse - torch.log(total)).abs() <= delta + 2.0 ** -22 * torch.log(total)).all()), part[0]


RATIO = 2.0 / (1 + 2.0 ** -8)  # of the two weights below: relative to the larger, the smaller lies between two bf16 numbers


def two_weights(n):
    """(sum of weights, sum of weights times values, sum of sizes) over the first i keys, i = 1 .. n; keys by turns weigh 1
    with value 2 and RATIO with value -1, so that nearly nothing is left of a mean."""
    p = torch.ones(n, dtype=torch.float64)
    p[1::2] = RATIO
    v = torch.full((n,), 2.0, dtype=torch.float64)
    v[1::2] = -1.0
    return p.cumsum(0), (p * v).cumsum(0), (p * v.abs()).cumsum(0)


def bits_tolerance(seen, total, sums, sizes, dt):
    """A weight in fp16 is off by 2^-11 at most, whatever the queries' type; sums and scores as elsewhere; then one rounding."""
    d = tolerances(seen, dt)[0]
    tol = (2.0 ** -11 + 2 * d) * sizes / total
    return tol + torch.finfo(dt).eps / 2 * ((sums / total).abs() + tol)


def test_the_tolerance_sees_weights_in_bf16():
    total, sums, sizes = (t[776] for t in two_weights(777))
    n1, n2 = 389, 388
    small = float(torch.tensor(256 / RATIO).bfloat16()) / 256 * RATIO  # the weight of 1 as bf16 would have it
    assert abs(small - 1) > 2.0 ** -9
    got = (n1 * small * 2.0 - n2 * RATIO) / float(total)
    for dt in (BF16, F16):
        assert abs(got - float(sums / total)) > float(bits_tolerance(777, total, sums, sizes, dt))


@gpu
@pytest.mark.parametrize("h,kv,d,dv,n,new,dt", [
    (8, 2, 128, 128, 777, 1, BF16), (8, 2, 128, 128, 777, 1, F16), (4, 1, 64, 64, 9001, 1, BF16), (16, 16, 192, 128, 500, 77, BF16),
    (8, 1, 256, 256, 300, 40, BF16), (512, 2, 128, 128, 270, 260, BF16), (512, 2, 64, 64, 270, 260, F16)])
def test_probabilities_have_eleven_bits(hip_device, h, kv, d, dv, n, new, dt):
    """(512 heads on 2 and 260 tokens: 64 rows a wave)"""
    from table_moe.ops import Fp8KVCache

    dev, page = hip_device, 64
    pages = -(-n // page)
    cache = Fp8KVCache(pages, kv, d, dv, page, device=dev)
    k, v = torch.zeros(n, kv, d), torch.full((n, kv, dv), 2.0)
    k[1::2, :, 5] = 1.0
    v[1::2] = -1.0
    table, lengths = torch.arange(pages, dtype=torch.int32, device=dev)[None], torch.tensor([n], dtype=torch.int32, device=dev)
    cache.append(k.to(dev), v.to(dev), table, lengths, torch.tensor([0, n], device=dev))
    q = torch.zeros(new, h, d, dtype=dt, device=dev)
    q[..., 5] = 1
    starts = None if new == 1 else torch.tensor([0, new], dtype=torch.int32, device=dev)
    y, lse = cache.attend(q, table, lengths, starts, scale=math.log(RATIO), return_lse=True)
    total, sums, sizes = (t[n - new:] for t in two_weights(n))
    tol = bits_tolerance(n, total, sums, sizes, dt)
    assert bool(((y.cpu().double() - (sums / total)[:, None, None]).abs() <= tol[:, None, None]).all())
    delta = tolerances(n, dt)[0]
    assert bool(((lse.cpu().double() - torch.log(total)[:, None]).abs() <= delta + 2.0 ** -22 * torch.log(total)[:, None]).all())

"""Rows of zeros and of non-finite values alone in the 8-bit cache: they ask for no scale, in a page that holds values and
in one that they begin."""

import math

import pytest
import torch

import kv8_ref as R
from test_gpu_kv8 import BF16, F16, F32, same_cells

pytestmark = pytest.mark.gpu


def append(cells, scale, rows, page_no, lo, hi):
    """The rule on one page [heads, page, D] of plain cells: rows [hi - lo, heads, D] at [lo, hi), in place."""
    for h in range(cells.shape[1]):
        x = rows[:, h].double()
        fin = x[torch.isfinite(x)].abs()
        top, was = float(fin.max()) if fin.numel() else 0.0, float(scale[page_no, h])
        held = cells[page_no, h, :lo]
        s = R.scale_of(top)
        if lo > 0 and top == 0:
            s = was
        elif lo > 0 and (was != 1 or bool((torch.nan_to_num(held) != 0).any())):
            s = max(s, was)
            if s != was:
                cells[page_no, h, :lo] = R.e4m3(held * (was / s))
        cells[page_no, h, lo:hi] = R.e4m3(x / s)
        scale[page_no, h] = s


def run(dev, page, d, dv, dt, steps, garbage):
    """steps: (tokens, function of (tokens, heads, columns) giving the rows) one after the other into one page."""
    from table_moe.ops import Fp8KVCache

    heads = 2
    cache = Fp8KVCache(3, heads, d, dv, page, device=dev)
    g = torch.Generator().manual_seed(5)
    if garbage:  # what another sequence left in the page
        for t in (cache.k, cache.v):
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g).to(torch.uint8))
    kc, vc = R.raw(cache.k, False), R.raw(cache.v, True)
    ks, vs = cache.k_scale.cpu().double(), cache.v_scale.cpu().double()
    table, at = torch.tensor([[1]], dtype=torch.int32, device=dev), 0
    for n, rows in steps:
        k, v = rows(g, n, heads, d).to(dt), rows(g, n, heads, dv).to(dt)
        cache.append(k.to(dev), v.to(dev), table, torch.tensor([at + n], device=dev), torch.tensor([0, n], device=dev))
        append(kc, ks, k, 1, at, at + n)
        append(vc, vs, v, 1, at, at + n)
        at += n
        assert torch.equal(cache.k_scale.cpu().double(), ks) and torch.equal(cache.v_scale.cpu().double(), vs), (n, at)
        same_cells(cache.k, kc, False)
        same_cells(cache.v, vc, True)
    return cache, ks, vs


def randn(size):
    return lambda g, n, h, d: size * torch.randn(n, h, d, generator=g)


def all_of(value):
    return lambda g, n, h, d: torch.full((n, h, d), value)


def one_small(g, n, h, d):
    """Zeros, but for the last token's last column."""
    x = torch.zeros(n, h, d)
    x[-1, :, -1] = 300.0  # its page's scale is 1
    return x


def one_first(g, n, h, d):
    x = torch.zeros(n, h, d)
    x[0, 0, 0] = -300.0
    return x


SHAPES = [(64, 128, 128, BF16), (32, 64, 64, F16), (128, 192, 128, F32), (64, 256, 256, BF16), (128, 192, 192, F16)]


@pytest.mark.parametrize("page,d,dv,dt", SHAPES)
@pytest.mark.parametrize("kind", [0.0, math.nan, math.inf])
def test_rows_without_values_after_small_tokens(hip_device, page, d, dv, dt, kind):
    """20 tokens of size 1e-3 keep their scale and their bytes; later small tokens get that scale, too."""
    cache, ks, vs = run(hip_device, page, d, dv, dt, [(20, randn(1e-3)), (1, all_of(kind)), (3, all_of(kind)), (4, randn(1e-3))],
                        garbage=True)
    assert float(ks[1].max()) < 2.0 ** -14 and float(vs[1].max()) < 2.0 ** -14


@pytest.mark.parametrize("page,d,dv,dt", SHAPES)
@pytest.mark.parametrize("first", [1, 4, 5, 31])
@pytest.mark.parametrize("kind", [0.0, math.nan])
def test_rows_without_values_at_the_start_of_a_page(hip_device, page, d, dv, dt, first, kind):
    """A page that begins with such rows takes the scale of the first values, whatever lies behind them in its storage."""
    page = max(page, 64) if first == 31 else page
    run(hip_device, page, d, dv, dt, [(first, all_of(kind)), (1, all_of(0.0)), (1, randn(1e-3)), (2, all_of(0.0)),
                                      (3, randn(1e-2))] if first < 31 else
        [(first, all_of(kind)), (2, randn(1e-3)), (6, randn(1e-4)), (5, randn(1.0))], garbage=True)


@pytest.mark.parametrize("page,d,dv,dt", SHAPES)
@pytest.mark.parametrize("held", [one_small, one_first])
@pytest.mark.parametrize("lo", [1, 3, 9, 30])
def test_a_page_whose_scale_is_1_for_a_value(hip_device, page, d, dv, dt, held, lo):
    """One value of 300 in one head or all, at the first or last cell: its scale of 1 binds the small rows that follow."""
    if held is one_small:
        _, ks, vs = run(hip_device, page, d, dv, dt, [(lo, one_small), (2, randn(1e-3))], garbage=True)
        assert bool((ks[1] == 1).all()) and bool((vs[1] == 1).all())
    else:
        _, ks, vs = run(hip_device, page, d, dv, dt, [(lo, one_first), (2, randn(1e-3))], garbage=True)
        assert float(ks[1, 0]) == 1 and float(ks[1, 1]) < 2.0 ** -14 and float(vs[1, 0]) == 1


def test_attention_over_a_page_with_a_zero_row(hip_device):
    """The small values' error stays that of 8 bits (half a step of e4m3, 2^-4, of each value)."""
    from table_moe.ops import Fp8KVCache

    g = torch.Generator().manual_seed(6)
    dev, d = hip_device, 64
    cache = Fp8KVCache(1, 1, d, page_size=64, device=dev)
    k, v = torch.randn(21, 1, d, generator=g), 1e-3 * torch.randn(21, 1, d, generator=g)
    k[20], v[20] = 0, 0
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    for n, rows in ((20, slice(0, 20)), (21, slice(20, 21))):
        cache.append(k[rows].to(dev), v[rows].to(dev), table, torch.tensor([n], device=dev),
                     torch.tensor([0, rows.stop - rows.start], device=dev))
    vd = cache.read_pages()[1][0, 0, :21].cpu()
    # (under 2^-6 of the scale a step is 2^-9 of it)
    scale = float(cache.v_scale[0, 0])
    assert bool(((vd - v[:, 0]).abs() <= v[:, 0].abs() * 2.0 ** -4 + scale * 2.0 ** -10).all()) and scale < 2.0 ** -14


@pytest.mark.parametrize("kind", [0.0, math.nan])
def test_storage_of_zeros_that_a_length_counts_as_held(hip_device, kind):
    """A wrapped pool of zeros, scales too, in a page of which a length says that it held tokens: zeros stay zeros."""
    from table_moe.ops import Fp8KVCache

    dev, d = hip_device, 64
    c = Fp8KVCache(2, 1, d, page_size=32, device=dev)
    z = lambda t: torch.zeros_like(t.view(torch.uint8)).view(t.dtype)  # noqa: E731
    w = Fp8KVCache.wrap(z(c.k), z(c.v), torch.zeros_like(c.k_scale), torch.zeros_like(c.v_scale))
    table, rows = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.full((3, 1, d), kind, device=dev)
    rows[1] = 0
    w.append(rows, rows, table, torch.tensor([8], device=dev), torch.tensor([0, 3], device=dev))
    for x in w.read_pages():
        bad = torch.isnan(x[0, 0])
        assert bool((x[0, 0][~bad] == 0).all())
        assert bad.any(1).nonzero().flatten().tolist() == ([] if kind == 0 else [5, 7])
    assert float(w.k_scale[0, 0]) == 1

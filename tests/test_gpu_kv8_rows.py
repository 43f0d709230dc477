"""Importance over the 8-bit cache by row of a call's new tokens, which is what the keep rule takes: pieces of prompts,
shared prefixes, packed sequences."""

import math

import pytest
import torch

import kv8_ref as R
from test_gpu_kv8 import BF16, F16, check_importance, filled, table_of

pytestmark = pytest.mark.gpu


def batch(g, lens, new, page, kv, d, dev, spare=1):
    counts = [-(-x // page) for x in lens]
    cache, plain = filled(g, sum(counts) + 2, kv, page, d, 128 if d == 192 else d, dev)
    table = table_of(g, counts, max(counts) + spare, sum(counts) + 2)
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    return cache, plain, table, torch.tensor(lens, dtype=torch.int32), starts


def by_rows(full, lens, new, rows):
    """The new tokens' part of [B, positions], packed; other rows 0."""
    out, first = full.new_zeros(rows), 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            if 0 <= n - m + i < full.shape[1]:
                out[first + i] = full[b, n - m + i]
        first += m
    return out


@pytest.mark.parametrize("page,h,kv,d,lens,new,dt", [
    (64, 32, 4, 128, [300, 70, 200], [37, 70, 1], BF16),        # a piece, a whole prompt, one token
    (32, 8, 2, 64, [500, 129, 64, 33], [200, 0, 33, 33], F16),   # none of one sequence
    (128, 12, 1, 64, [1200], [700], BF16),                       # several workgroups a sequence, one key head
    (64, 16, 16, 192, [95, 96, 97], [31, 32, 33], F16),
    (32, 40, 1, 256, [40, 65], [3, 64], BF16),
])
@pytest.mark.parametrize("with_lse", [False, True])
def test_importance_of_new_tokens(hip_device, page, h, kv, d, lens, new, dt, with_lse):
    g = torch.Generator().manual_seed(h + d + sum(new))
    dev = hip_device
    cache, plain, table, lengths, starts = batch(g, lens, new, page, kv, d, dev)
    q = (1.5 * torch.randn(len(lens), h, d, generator=g)).to(dt)
    args = (q.to(dev), table.to(dev), lengths.to(dev))
    lse = cache.attend(*args, return_lse=True)[1] if with_lse else None
    full = cache.importance(*args, lse=lse)
    check_importance(plain, q, table, lengths, d ** -0.5, full)
    rows = sum(new) + 3  # (rows of no sequence behind the last one)
    got = cache.importance(*args, lse=lse, starts=starts.to(dev), out_len=rows)
    assert got.shape == (rows,) and torch.equal(got.cpu(), by_rows(full.cpu(), lens, new, rows))
    again = cache.importance(*args, lse=lse, starts=starts.long().to(dev), out_len=rows)
    assert torch.equal(got, again)


def test_keep_rule_of_pieces_and_packed_sequences(hip_device):
    """cached_importance through build_prefill_keep_mask: a piece behind a prefix, a whole prompt and a short piece, packed.
    The kept experts are those of the scores in 64 bits, not those of the prefix's."""
    from table_moe.skip.pruning import build_prefill_keep_mask
    from table_moe.utils import ModalityContext
    from table_moe.utils.importance import cached_importance

    g = torch.Generator().manual_seed(42)
    dev, page, h, kv, d, e = hip_device, 64, 8, 2, 128, 24
    lens, new = [260, 50, 130], [60, 50, 20]
    cache, plain, table, lengths, starts = batch(g, lens, new, page, kv, d, dev)
    n = sum(new)
    q = (2 * torch.randn(n, h, d, generator=g)).to(BF16)
    last = starts[1:].long() - 1
    _, lse = cache.attend(q.to(dev), table.to(dev), lengths.to(dev), starts.to(dev), return_lse=True)
    got = cached_importance(cache, q[last].to(dev), table.to(dev), lengths.to(dev), lse=lse[last.to(dev)], query_length=n,
                            starts=starts.to(dev))
    assert got.shape == (n,) and ModalityContext.get_attn_weights() is not None
    k = plain[0] * plain[1][:, :, None, None]
    want, tol = [], 0.0
    for b, (length, m) in enumerate(zip(lens, new)):
        kk = R.sequence(k, table, b, length)
        _, _, _, size, p = R.attend(q[last[b]].double(), kk, kk, torch.ones(length, dtype=torch.bool), d ** -0.5)
        want.append(p.mean(1)[length - m:])
        # as in check_importance: the score's error and the sum's, relative
        tol = max(tol, 4 * (float(size.max()) * (2 * d * 2.0 ** -24 + 3 * 2.0 ** -23) + 2.0 ** -21 + length * 2.0 ** -24))
    want = torch.cat(want)
    assert bool(((got.cpu().double() - want).abs() <= tol * want).all())
    sel = torch.stack([torch.randperm(e, generator=g)[:4] for _ in range(n)])
    w = torch.rand(n, 4, generator=g)
    keep = build_prefill_keep_mask(sel.to(dev), w.to(dev), ModalityContext.get_attn_weights(), e, 0.5).cpu()
    score = torch.zeros(e, dtype=torch.float64).index_add_(0, sel.reshape(-1), (w.double() * want[:, None]).reshape(-1))
    order = score.argsort(descending=True)
    gap = score[order[e // 2 - 1]] / score[order[e // 2]] - 1
    assert float(gap) > 3 * tol  # (each sum's own error is under tol)
    kept = torch.zeros(e, dtype=torch.bool)
    kept[order[:e // 2]] = True
    assert torch.equal(keep, kept[sel])
    # without a prefix the rows are the positions
    one = cached_importance(cache, q[last[1:2]].to(dev), table[1:2].to(dev), lengths[1:2].to(dev), query_length=50)
    two = cached_importance(cache, q[last[1:2]].to(dev), table[1:2].to(dev), lengths[1:2].to(dev), query_length=50,
                            starts=torch.tensor([0, 50], device=dev))
    assert torch.equal(one.reshape(-1), two)
    # the same as the function over 16-bit keys, whose query_length are the last ones
    from table_moe.utils.importance import cache_last_token_attention

    keys = cache.read_pages(table[0, :-(-260 // page)].long().to(dev))[0].transpose(1, 2).flatten(0, 1)[:260].to(BF16)
    over16 = cache_last_token_attention(q[None, :60].to(dev), keys[None], d ** -0.5, None, 60)
    assert bool(((over16.reshape(-1).cpu().double() - want[:60]).abs() <= tol * want[:60]).all())


def test_importance_rows_of_odd_batches(hip_device):
    """Pages that are not there, more new tokens than positions, positions past the table, lists that make no sense, no rows."""
    g = torch.Generator().manual_seed(42)
    dev, page, d = hip_device, 32, 64
    cache, plain = filled(g, 8, 2, page, d, d, dev)
    table = torch.tensor([[0, 99, 1], [2, 3, -4], [4, 5, 6]], dtype=torch.int32, device=dev)
    lens, new = [90, 20, 200], [60, 30, 150]
    q = torch.randn(3, 8, d, generator=g).to(BF16).to(dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    starts = torch.tensor([0, 60, 90, 240], dtype=torch.int32, device=dev)
    full = cache.importance(q, table, lengths)
    got = cache.importance(q, table, lengths, starts=starts, out_len=240)
    assert torch.equal(got.cpu(), by_rows(full.cpu(), lens, new, 240))
    assert bool((got[2:34] == 0).all()) and bool((got[60:70] == 0).all()) and float(got[34:60].min()) > 0
    for bad in ([0, 1 << 30, -5, 7], [9, 3, 2, 1], [5, 5, 5, 5]):  # in bounds, whatever they say
        y = cache.importance(q, table, lengths, starts=torch.tensor(bad, dtype=torch.int32, device=dev), out_len=11)
        assert y.shape == (11,) and bool(torch.isfinite(y).all())
    assert cache.importance(q, table, lengths, starts=starts, out_len=0).shape == (0,)
    assert cache.importance(q[:0], table[:0], lengths[:0], starts=starts[:1], out_len=4).tolist() == [0.0] * 4


def test_importance_rows_captured(hip_device):
    """One captured call, replayed over other lengths and starts between eager work."""
    g = torch.Generator().manual_seed(43)
    dev, page, d, kv = hip_device, 64, 64, 2
    cache, plain, table, lengths, starts = batch(g, [400, 300], [30, 40], page, kv, d, dev)
    q, table, lengths, starts = ((t.to(dev)) for t in (torch.randn(2, 8, d, generator=g).to(BF16), table, lengths, starts))
    call = lambda: cache.importance(q, table, lengths, starts=starts, out_len=70)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for lens, cut in (([400, 300], 30), ([100, 299], 1), ([399, 70], 60), ([65, 33], 0)):
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        starts.copy_(torch.tensor([0, cut, 70], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call())
        torch.cuda.synchronize()


def test_importance_rows_refusals(hip_device):
    from table_moe.ops import Fp8KVCache
    from table_moe.utils.importance import cached_importance

    dev = hip_device
    c = Fp8KVCache(4, 2, 128, device=dev)
    q = torch.zeros(3, 4, 128, dtype=BF16, device=dev)
    t, n = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    s = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
    assert c.importance(q, t, n, starts=s, out_len=3).shape == (3,)
    for kw in (dict(out_len=None), dict(out_len=-1), dict(starts=s[:3]), dict(starts=s.float()), dict(starts=s[None]),
               dict(scale=math.nan), dict(lse=torch.zeros(3, 3, device=dev))):
        with pytest.raises(ValueError):
            c.importance(q, t, n, **{**dict(starts=s, out_len=3), **kw})
    with pytest.raises(ValueError):
        c.importance(q[:2], t, n, starts=s, out_len=3)
    with pytest.raises(ValueError):
        cached_importance(c, q, t, n, starts=s)

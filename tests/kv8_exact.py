"""Inputs for attention over the 8-bit cache whose scores are whole numbers and whose probabilities are powers of two, so
that what a result may be off by is a few roundings, and a tile or a key that is lost or counted twice shows.

K holds whole numbers from -2 to 2, a query four entries of 1 or -1 (each head its own columns), the scale is ln 2: a key's
weight is 2^s with a whole s from -8 to 8, exact in fp16.  V names tiles: tile t (over all sequences) has its keys' values, 1
to 7, in column t % v_dim, and 0 elsewhere."""

import math

import torch

import kv8_ref as R

LN2 = math.log(2.0)


def table_for(g, lens, page, spare=2):
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table, at = torch.full((len(lens), max(counts) + 1), -1, dtype=torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pages


class Inputs:
    def __init__(self, seed, page, h, kv, d, dv, lens, new, dt):
        g = torch.Generator().manual_seed(seed)
        self.page, self.h, self.kv, self.d, self.dv, self.lens, self.dt = page, h, kv, d, dv, lens, dt
        self.new = [1] * len(lens) if new is None else new
        self.table, self.pages = table_for(g, lens, page)
        self.lengths = torch.tensor(lens, dtype=torch.int32)
        self.starts = None if new is None else torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
        n = sum(self.new)
        # whole numbers per sequence [n, kv, d]
        self.k = [torch.randint(-2, 3, (m, kv, d), generator=g).double() for m in lens]
        self.value = [torch.randint(1, 8, (m, kv), generator=g).double() for m in lens]
        self.q = torch.zeros(n, h, d, dtype=torch.float64)
        at = torch.argsort(torch.rand(n, h, d, generator=g), -1)[..., :4]
        self.q.scatter_(2, at, torch.randint(0, 2, (n, h, 4), generator=g).double() * 2 - 1)
        first = torch.tensor([0, *[-(-m // 32) for m in lens]]).cumsum(0)
        self.tile0 = first[:-1].tolist()  # each sequence's first tile over all
        self.ks = 2.0 ** torch.randint(-1, 3, (self.pages, kv), generator=g).double()
        self.vs = 2.0 ** torch.randint(-2, 3, (self.pages, kv), generator=g).double()

    def column(self, b, keys):
        return (self.tile0[b] + keys // 32) % self.dv

    def pages_of(self, rows, scale, spare):
        """Plain cells [pages, kv, page, columns] of values by sequence; pages of nobody and cells past an end hold `spare`."""
        cols = rows[0].shape[2]
        cells = torch.full((self.pages, self.kv, self.page, cols), float(spare), dtype=torch.float64)
        for b, x in enumerate(rows):
            for p in range(-(-len(x) // self.page)):
                part = x[p * self.page:(p + 1) * self.page].transpose(0, 1)
                cells[self.table[b, p], :, :part.shape[1]] = part / scale[self.table[b, p]][:, None, None]
        return cells

    def values(self):
        out = []
        for b, w in enumerate(self.value):
            v = torch.zeros(len(w), self.kv, self.dv, dtype=torch.float64)
            if len(w):
                keys = torch.arange(len(w))
                v[keys, :, self.column(b, keys)] = w
            out.append(v)
        return out

    def cache(self, dev, k=None, v=None):
        from table_moe.ops import Fp8KVCache

        c = Fp8KVCache(self.pages, self.kv, self.d, self.dv, self.page, device=dev)
        for packed, rows, scale, to, values in ((c.k, self.k if k is None else k, self.ks, c.k_scale, False),
                                                (c.v, self.values() if v is None else v, self.vs, c.v_scale, True)):
            cells = self.pages_of(rows, scale, 160.0)
            assert torch.equal(R.e4m3(cells), cells)
            packed.view(torch.uint8).copy_(R.pack(cells, values).view(torch.uint8))
            to.copy_(scale.float())
        return c

    def args(self, dev):
        return (self.table.to(dev), self.lengths.to(dev)) + (() if self.starts is None else (self.starts.to(dev),))

    def rows(self):
        """(row, sequence, number of keys that it sees with causal masks)"""
        r = 0
        for b, (n, m) in enumerate(zip(self.lens, self.new)):
            for i in range(m):
                yield r, b, max(0, n - m + i + 1)
                r += 1

    def weights(self, row, b, seen):
        """2^s [seen, heads] of a row."""
        k = self.k[b][:seen].repeat_interleave(self.h // self.kv, 1)
        return torch.exp2(torch.einsum("hd,nhd->nh", self.q[row], k))

    def tiles(self, row, b, seen, first=0):
        """(sum of weights [tiles, heads], sum of weights times values): tiles of 32 keys from `first` on."""
        p = self.weights(row, b, seen)
        n = -(-seen // 32)
        pad = lambda x: torch.cat([x, x.new_zeros(n * 32 - seen, self.h)]).view(n, 32, self.h).sum(1)  # noqa: E731
        return pad(p), pad(p * self.value[b][:seen].repeat_interleave(self.h // self.kv, 1))


def by_column(inp, b, w):
    """[tiles, heads] -> [heads, v_dim]: each tile's share in its column."""
    y = torch.zeros(inp.dv, inp.h, dtype=torch.float64)
    y.index_add_(0, inp.column(b, 32 * torch.arange(len(w))), w)
    return y.T


def tolerances(seen, dt):
    """(relative error of a sum of probabilities, or of them with values; half a step of the result's type).

    The scale ln 2 and log2 e are rounded, and so is their product: 3 x 2^-24 of |s| <= 8; s times that plus an offset is
    rounded twice, |s| + |m| <= 40 (a reference is up to 2^8 under the row's largest, a value's scale up to 2^2): 2 x 40 x
    2^-24; all times ln 2, and once more for the other side of the quotient.  An exponential: 2^-22.  Sums: a lane adds 16,
    then its wave's tiles in a part, then the halves, four waves and up to 128 parts; products add 32 at a time.  A part has
    at most max(seen / 4 waves, ...) keys: seen / 128 + 16 + 134 roundings of 2^-24 where tiles are added one by one."""
    d = 2 * math.log(2) * (3 * 8 + 2 * 40) * 2.0 ** -24 + 2.0 ** -21 + (seen / 128 + 150) * 2.0 ** -24
    return d, torch.finfo(dt).eps / 2


def accepts(y, lse, sums, total, seen, dt):
    """Whether y [.., heads, v_dim] and lse [.., heads] are sums / total and log total, up to the roundings."""
    d, u = tolerances(seen, dt)
    want, wl = sums / total[..., None], torch.log(total)
    ok = ((y - want).abs() <= 2 * d * want.abs() * (1 + u) + u * want.abs() + (2.0 ** -25 if dt == torch.float16 else 0)).all(-1)
    return ok & ((lse - wl).abs() <= d + 2.0 ** -22 * wl.abs())

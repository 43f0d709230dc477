"""The 8-bit cache's definition in 64 bits on the host, from its documented
layout and rules (no code of the package)."""

import math

import torch

MAX = 448.0


def scale_of(amax: float) -> float:
    """Smallest power of two s >= 2^-100 with amax / s <= 448; 1 for 0."""
    if amax == 0:
        return 1.0
    e = -100
    f = math.frexp(amax)  # amax = f[0] 2^f[1]
    e = max(e, f[1] - 9 - 1)
    while amax / 2.0 ** e > MAX:
        e += 1
    return 2.0 ** e


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value (ties to even) of |v| <= 448; NaN where v is not finite."""
    a = v.abs()
    step = torch.exp2(torch.clamp(torch.frexp(torch.where(torch.isfinite(a), a, torch.zeros_like(a))).exponent.double() - 1,
                                  min=-6.0) - 3.0)
    r = torch.sign(v) * torch.round(a / step) * step
    return torch.where(torch.isfinite(v), r, torch.full_like(v, math.nan))


def cells(page: int, d: int, values: bool):
    """(token, column) of each byte of a page."""
    t = torch.arange(page // 32).view(-1, 1, 1, 1)
    j = torch.arange(d // 32).view(1, -1, 1, 1)
    lane = torch.arange(64).view(1, 1, -1, 1)
    e = torch.arange(16).view(1, 1, 1, -1)
    if values:
        token, col = 16 * (e // 8) + 8 * (e // 4 % 2) + 4 * (lane // 32) + e % 4, 32 * j + lane % 32
    else:
        token, col = lane % 32, 32 * j + 16 * (lane // 32) + e
    shape = (page // 32, d // 32, 64, 16)
    return (32 * t + token).expand(shape), col.expand(shape)


def raw(packed: torch.Tensor, values: bool) -> torch.Tensor:
    """[pages, heads, page, D] float64 of a packed tensor's bytes as numbers."""
    p, h, tiles, blocks = packed.shape[:4]
    token, col = cells(tiles * 32, blocks * 32, values)
    out = torch.zeros(p, h, tiles * 32, blocks * 32, dtype=torch.float64)
    out[:, :, token, col] = packed.cpu().float().double()
    return out


def pack(x: torch.Tensor, values: bool) -> torch.Tensor:
    token, col = cells(x.shape[2], x.shape[3], values)
    return x[:, :, token, col].float().to(torch.float8_e4m3fn)


def append(cells_, scale, rows, table, lengths, starts):
    """The rule of append on plain cells [pages, heads, page, D] and scales, in place."""
    page = cells_.shape[2]
    for b in range(len(lengths)):
        first, end = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        old = int(lengths[b]) - (end - first)
        for p in range(table.shape[1]):
            lo, hi = max(old, p * page, 0), min(int(lengths[b]), (p + 1) * page)
            at = int(table[b, p])
            if lo >= hi or end == first or not 0 <= at < cells_.shape[0]:
                continue
            new = rows[first + lo - old:first + hi - old].double()  # [m, heads, D]
            for h in range(cells_.shape[1]):
                x = new[:, h]
                fin = x[torch.isfinite(x)].abs()
                s = scale_of(float(fin.max()) if fin.numel() else 0.0)
                was = float(scale[at, h])
                if lo > p * page:
                    s = max(s, was)
                    held = cells_[at, h, :lo - p * page]
                    if s != was:
                        cells_[at, h, :lo - p * page] = e4m3(held * (was / s))
                cells_[at, h, lo - p * page:hi - p * page] = e4m3(x / s)
                scale[at, h] = s


def sequence(values, table, b, n):
    """Positions [0, n) of a sequence [n, heads, D]."""
    page = values.shape[2]
    ids = [int(table[b, p]) for p in range(-(-n // page))]
    return torch.cat([values[i].transpose(0, 1) for i in ids])[:n] if ids else values.new_zeros(0, *values.shape[1::2])


def attend(q, k, v, visible, scale):
    """q [H, D], k [n, Hkv, D], v [n, Hkv, Dv], visible [n] -> (y [H, Dv], lse [H], sum p |v|, sum |q k| scale, p)."""
    g = q.shape[0] // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1)[visible], v.repeat_interleave(g, 1)[visible]
    if kk.shape[0] == 0:
        z = q.new_zeros(q.shape[0], v.shape[2])
        return z, torch.full((q.shape[0],), -math.inf, dtype=q.dtype), z, q.new_zeros(q.shape[0]), q.new_zeros(0, q.shape[0])
    s = torch.einsum("hd,nhd->nh", q, kk) * scale
    size = torch.einsum("hd,nhd->nh", q.abs(), kk.abs()).amax(0) * scale
    p = torch.softmax(s, 0)
    return torch.einsum("nh,nhd->hd", p, vv), torch.logsumexp(s, 0), torch.einsum("nh,nhd->hd", p, vv.abs()), size, p

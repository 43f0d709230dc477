"""The attention side of a cached MoE layer, as measurable cases.

Queries and keys are rotated by positions of several axes (time, height, width),
keys and values are written into a paged cache that holds them in 8 bits (e4m3)
with one fp32 scale per page and head, attention reads that cache, and so does
the importance of the prompt's tokens, from which the layer's keep rule goes.
The kinds below are these four calls.

Heads are those of the two model families of the tests and the benchmark (32
query heads on 4 key heads of 128; 16 heads of 192 with values of 128) or
generic ones.

The cache: tiles of 32 tokens.  k [pages, heads, page / 32, D / 32, 64, 16]: byte
e of lane l of column block j is token l % 32 of the tile, column 32 j + 16 (l /
32) + e.  v of the same shape over its own columns: column 32 j + l % 32, token
16 (e / 8) + 8 (e / 4 % 2) + 4 (l / 32) + e % 4.  Scales [pages, heads].  A batch:
table [sequences, most pages] of page numbers, lengths [sequences] with the new
tokens counted, starts [sequences + 1]: where each sequence's new tokens begin
(None: one each).
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
THETA = 5000000.0


def _ops():
    if not hasattr(_ops, "module"):  # imported once, as a user's program does
        root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "tablemoe-sc26_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        from table_moe import ops

        _ops.module = ops
    return _ops.module


# --------------------------------------------------------------------- cases
def _rotate(name, n, heads, kv, dim, turned, sections, far, dtype, interleaved=False, adjacent=False, inverse=False):
    return dict(name=name, kind="rotate", n=n, heads=heads, kv=kv, dim=dim, turned=turned, sections=sections, far=far,
                dtype=dtype, interleaved=interleaved, adjacent=adjacent, inverse=inverse)


def _batch(name, kind, seqs, context, new, heads, kv, dim, vdim, page, dtype, **more):
    return dict(name=name, kind=kind, seqs=seqs, context=context, new=new, heads=heads, kv=kv, dim=dim, vdim=vdim,
                page=page, dtype=dtype, **more)


def listed():
    return [
        # one decode step of a small batch, far into its contexts
        _rotate("rotate_decode_8", 8, 32, 4, 128, 128, "24,20,20", 100000, "bf16", interleaved=True),
        # a prompt of text and images
        _rotate("rotate_prefill_4099", 4099, 32, 4, 128, 128, "24,20,20", 0, "bf16", interleaved=True),
        # the gradient of a long video's rotation, the axes' frequencies in runs
        _rotate("rotate_back_video_30011", 30011, 32, 4, 128, 128, "16,24,24", 0, "f16", inverse=True),
        # the tokens of one decode step, into pages that are partly full
        _batch("append_decode_32", "append", 32, 8192, 1, 32, 4, 128, 128, 64, "bf16"),
        # several prompts at once
        _batch("append_prompts_3", "append", 3, 4500, 4500, 32, 4, 128, 128, 64, "f16"),
        # one token after a short prompt: latency
        _batch("attend_decode_1", "attend", 1, 777, 1, 32, 4, 128, 128, 64, "bf16", causal=True, lse=False),
        # a decode step of a batch with contexts of many lengths
        _batch("attend_decode_32", "attend", 32, 8192, 1, 32, 4, 128, 128, 64, "bf16", causal=True, lse=False),
        # one token at the end of a long video
        _batch("attend_decode_131071", "attend", 1, 131071, 1, 32, 4, 128, 128, 64, "f16", causal=True, lse=True),
        # a prompt over its own tokens
        _batch("attend_prefill_4099", "attend", 1, 4099, 4099, 32, 4, 128, 128, 64, "bf16", causal=True, lse=True),
        # pieces of long prompts, a key head for each query head, values narrower than keys
        _batch("attend_piece_9000", "attend", 3, 9000, 1024, 16, 16, 192, 128, 64, "f16", causal=True, lse=False),
        # the prompt's importance for the keep rule
        _batch("importance_4099", "importance", 1, 4099, 1, 32, 4, 128, 128, 64, "bf16", lse=False),
        # a long video's, with the attention's normaliser at hand
        _batch("importance_131071", "importance", 1, 131071, 1, 32, 4, 128, 128, 64, "bf16", lse=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "append", "append", "attend", "attend", "attend", "attend", "importance",
                       "importance"])
    if kind == "rotate":
        dim = rng.choice([64, 128, 128, 192, 256])
        turned = rng.choice([dim, dim, dim // 2])
        axes = rng.choice([1, 2, 3, 3])
        half, cut = turned // 2, []
        left = half
        for a in range(axes - 1):
            cut.append(rng.randint(1, max(1, left // 2)))
            left -= cut[-1]
        heads, kv = rng.choice([(32, 4), (16, 16), (12, 2), (7, 1)])
        return dict(kind=kind, n=_log_int(rng, 1, 15000), heads=heads, kv=kv, dim=dim, turned=turned,
                    sections=",".join(map(str, [left, *cut])), far=rng.choice([0, 5000, 200000]),
                    dtype=rng.choice(["bf16", "f16", "f32"]), interleaved=rng.random() < 0.5,
                    adjacent=rng.random() < 0.3, inverse=rng.random() < 0.4)
    heads, kv, dim, vdim = rng.choice([(32, 4, 128, 128), (32, 4, 128, 128), (16, 16, 192, 128), (16, 2, 64, 64),
                                       (12, 4, 128, 128), (8, 1, 256, 256), (24, 8, 192, 192)])
    case = dict(kind=kind, heads=heads, kv=kv, dim=dim, vdim=vdim, page=rng.choice([32, 64, 64, 128]),
                dtype=rng.choice(["bf16", "f16"]))
    if kind == "append":
        seqs = _log_int(rng, 1, 32)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 12000 // seqs))
        case.update(seqs=seqs, new=new, context=new + _log_int(rng, 1, 4000), dtype=rng.choice(["bf16", "f16", "f32"]))
    elif kind == "importance":
        seqs = _log_int(rng, 1, 8)
        case.update(seqs=seqs, new=1, context=_log_int(rng, 1, 60000 // seqs), lse=rng.random() < 0.5)
    elif rng.random() < 0.6:  # single tokens, or a few that were drafted
        seqs = _log_int(rng, 1, 48)
        new = rng.choice([1, 1, 1, 4])
        case.update(seqs=seqs, new=new, context=new + _log_int(rng, 1, 200000 // seqs), causal=True,
                    lse=rng.random() < 0.5)
    else:
        seqs = _log_int(rng, 1, 6)
        new = _log_int(rng, 2, 3000 // seqs)
        case.update(seqs=seqs, new=new, context=new + rng.choice([0, _log_int(rng, 1, 4000)]),
                    causal=rng.random() < 0.8, lse=rng.random() < 0.5)
    return case


def _lens(case):
    """(lengths, new tokens) of the batch's sequences; the first has both as the case names them."""
    r = random.Random(case["context"] * 131 + case["seqs"])
    lens, new = [case["context"]], [case["new"]]
    for _ in range(case["seqs"] - 1):
        n = case["new"] if case["new"] <= 4 else r.randint(case["new"] // 2, case["new"])
        new.append(n)
        lens.append(n if case["new"] == case["context"] else max(n, r.randint(case["context"] // 8, case["context"])))
    return lens, new


# -------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    t = torch.randn(*shape, generator=g, device=DEV, dtype=dtype)
    return t if scale == 1.0 else t.mul_(scale)


def _heads(g, n, h, d, dt, scale=1.0):
    """Vectors of heads: a few channels are larger than the rest."""
    return (_randn(g, n, h, d) * torch.exp(0.4 * _randn(g, h, d)) * scale).to(dt)


def _prompt_positions(n, axes, far, r):
    """Positions of n tokens: runs of text (all axes alike), images and clips (frame, row and column)."""
    out, at = np.zeros((axes, n), dtype=np.int64), far
    i = 0
    while i < n:
        m = min(n - i, r.randint(20, 200))
        out[:, i:i + m] = at + np.arange(m)
        i, at = i + m, at + m
        t, h, w = r.choice([1, 1, 4, 8]), r.randint(6, 24), r.randint(6, 24)
        m = min(n - i, t * h * w)
        k = np.arange(m)
        grid = [k // (h * w), k // w % h, k % w]
        for a in range(axes):
            out[a, i:i + m] = at + (grid[a] if axes == 3 else grid[1 + a] if axes == 2 else k)
        i, at = i + m, at + (m if axes == 1 else max(t, h, w))
    return torch.from_numpy(out).to(DEV)


def _pow2_scale(amax):
    """The smallest power of two s >= 2^-100 with amax / s <= 448 (1 where amax is 0)."""
    m, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875)).clamp_min(-100)
    return torch.where(amax > 0, ((e + 127) << 23).to(torch.int32).view(torch.float32), torch.ones_like(amax))


def _pack_k(x):
    p, h, page, d = x.shape
    return x.view(p, h, page // 32, 32, d // 32, 2, 16).permute(0, 1, 2, 4, 5, 3, 6).reshape(
        p, h, page // 32, d // 32, 64, 16)


def _unpack_k(k):
    p, h, tiles, blocks = k.shape[:4]
    return k.view(p, h, tiles, blocks, 2, 32, 16).permute(0, 1, 2, 5, 3, 4, 6).reshape(p, h, tiles * 32, blocks * 32)


def _pack_v(x):
    p, h, page, d = x.shape
    return x.view(p, h, page // 32, 2, 2, 2, 4, d // 32, 32).permute(0, 1, 2, 7, 5, 8, 3, 4, 6).reshape(
        p, h, page // 32, d // 32, 64, 16)


def _unpack_v(v):
    p, h, tiles, blocks = v.shape[:4]
    return v.view(p, h, tiles, blocks, 2, 32, 2, 2, 4).permute(0, 1, 2, 6, 7, 4, 8, 3, 5).reshape(
        p, h, tiles * 32, blocks * 32)


def _filled(g, pages, case):
    """A pool of pages in use: (k, v, k_scale, v_scale)."""
    out = []
    for d, pack, size in ((case["dim"], _pack_k, 1.0), (case["vdim"], _pack_v, 0.7)):
        x = _randn(g, pages, case["kv"], case["page"], d, scale=size)
        x *= torch.exp(0.4 * _randn(g, case["kv"], 1, d)) * torch.exp(0.3 * _randn(g, pages, case["kv"], 1, 1))
        s = _pow2_scale(x.abs().amax((2, 3)))
        out.append((pack((x / s[:, :, None, None]).to(E4M3)).contiguous(), s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    dt = DTYPES[case["dtype"]]
    h, kv = case["heads"], case["kv"]
    if kind == "rotate":
        n, half = case["n"], case["turned"] // 2
        axes = case["sections"].count(",") + 1
        r = random.Random(seed)
        if case["far"] and n <= 64:  # one token of each of n sequences: text, all axes alike
            positions = torch.tensor([[r.randint(case["far"] // 2, case["far"]) for _ in range(n)]] * axes, device=DEV)
        else:
            positions = _prompt_positions(n, axes, case["far"], r)
        sections = np.array([int(v) for v in case["sections"].split(",")])
        i = np.arange(half)
        if case["interleaved"]:
            axis = np.where(i < sections[i % axes] * axes, i % axes, 0)
        else:
            axis = np.searchsorted(np.cumsum(sections), i, side="right")
        inv = (THETA ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(DEV)
        return dict(case=case, q=_heads(g, n, h, case["dim"], dt), k=_heads(g, n, kv, case["dim"], dt), inv=inv,
                    positions=positions, axis=torch.from_numpy(axis).to(DEV))  # axis: each frequency's
    lens, new = _lens(case)
    page = case["page"]
    counts = [-(-n // page) for n in lens]
    most, total = max(counts), sum(counts)
    order = torch.randperm(total + 3, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(case["seqs"], most, dtype=torch.int32, device=DEV)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    st = dict(case=case, cache=_filled(g, total + 3, case), table=table,
              lengths=torch.tensor(lens, dtype=torch.int32, device=DEV),
              starts=None if max(new) == 1 else torch.tensor(np.cumsum([0, *new]), dtype=torch.int32, device=DEV),
              most_new=max(new), most=max(lens))
    n = sum(new)
    if kind == "append":
        st.update(k=_heads(g, n, kv, case["dim"], dt), v=_heads(g, n, kv, case["vdim"], dt, 0.7))
        return st
    st["q"] = _heads(g, n, h, case["dim"], dt, 1.2)
    if kind == "importance" and case["lse"]:
        s = _scores(st["q"][:, None], st)  # [B, kv, rows, L]
        st["lse"] = torch.logsumexp(s, 3).view(case["seqs"], h).contiguous()
    return st


# ----------------------------------------------------------- the plain forms
def _rotate_plain(x, st, c):
    half = c["turned"] // 2
    angle = (st["positions"][st["axis"]].double() * st["inv"].double()[:, None]).T  # far positions: 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if c["inverse"]:
        sin = -sin
    y = x.float()
    if c["adjacent"]:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1).to(x.dtype)


def _where_new(st):
    """(sequence, number in it) of each new token."""
    t = torch.arange((st["k"] if "k" in st else st["q"]).shape[0], device=DEV)
    if st["starts"] is None:
        return t, torch.zeros_like(t)
    b = torch.searchsorted(st["starts"], t, right=True) - 1
    return b, t - st["starts"][b]


def _append_plain(x, packed, scale, pack, unpack, st):
    """Writes x [tokens, kv, D] into the pages that it touches: up to `many` of each sequence."""
    c = st["case"]
    page, seqs = c["page"], st["table"].shape[0]
    b, i = _where_new(st)
    new = torch.ones_like(st["lengths"]) if st["starts"] is None else st["starts"][1:] - st["starts"][:-1]
    old = st["lengths"] - new  # tokens held before
    many = (st["most_new"] + page - 2) // page + 1
    which = old[:, None] // page + torch.arange(many, device=DEV)
    last = (st["lengths"] - 1) // page
    which = torch.minimum(which, last[:, None])  # past the last page: that page again, with what it gets
    ids = st["table"].gather(1, which.long()).long()
    held = unpack(packed[ids.view(-1)]).float().view(seqs, many, c["kv"], page, -1)
    before = scale[ids]
    pos = old[b] + i
    at, cell = pos // page - old[b] // page, pos % page
    fresh = held.new_zeros(held.shape)
    fresh[b, at, :, cell] = x.float()
    s = _pow2_scale(fresh.abs().amax((3, 4)))
    s[:, 0] = torch.where((old % page > 0)[:, None], torch.maximum(s[:, 0], before[:, 0]), s[:, 0])
    place = which[..., None] * page + torch.arange(page, device=DEV)  # [B, many, page]: the cells' positions
    # what the pages held keeps its value as far as 8 bits can: rounded again where a scale rose
    was = (place < old[:, None, None])[:, :, None, :, None]
    now = (place < st["lengths"][:, None, None])[:, :, None, :, None] & ~was
    y = torch.where(was, held * (before / s)[..., None, None], torch.where(now, fresh / s[..., None, None], held))
    same = (which - which[:, :1]).long()  # the first of equal pages is the one that got the tokens
    y = y.gather(1, same[:, :, None, None, None].expand_as(y)).flatten(0, 1)
    s = s.gather(1, same[:, :, None].expand_as(s)).flatten(0, 1)
    packed.view(torch.uint8)[ids.view(-1)] = pack(y.to(E4M3)).view(torch.uint8)
    scale[ids.view(-1)] = s


def _pages(st, which):
    """Keys (0) or values (1) of every sequence, [B, kv, L, D] in 32 bits."""
    t = st["table"].long()
    x = (_unpack_k, _unpack_v)[which](st["cache"][which][t.view(-1)])  # [B * pages, kv, page, D]
    x = x.float() * st["cache"][2 + which][t.view(-1)][..., None, None]
    return x.view(*t.shape, *x.shape[1:]).transpose(1, 2).flatten(2, 3)


def _scores(q, st):
    """Scores [B, kv, tokens * heads of a key head, L] of q [B, tokens, H, D]; keys past the end: -inf."""
    c = st["case"]
    b, n, h, d = q.shape
    k = _pages(st, 0)
    rows = q.view(b, n, c["kv"], h // c["kv"], d).transpose(1, 2).reshape(b, c["kv"], -1, d).float()
    s = (rows @ k.mT.contiguous()) * d ** -0.5
    past = torch.arange(k.shape[2], device=DEV) >= st["lengths"][:, None]
    return s.masked_fill_(past[:, None, None], -math.inf)


def _attend_plain(q, st):
    c = st["case"]
    b, i = _where_new(st)
    n, h, d = q.shape
    seqs, kv, most = st["table"].shape[0], c["kv"], st["most_new"]
    padded = q.new_zeros(seqs, most, h, d)
    padded[b, i] = q
    s = _scores(padded, st)  # [B, kv, most * g, L]
    if c["causal"]:
        new = st["lengths"] * 0 + 1 if st["starts"] is None else st["starts"][1:] - st["starts"][:-1]
        last = (st["lengths"] - new)[:, None] + torch.arange(most, device=DEV)  # the last key that a token sees
        last = last.repeat_interleave(h // kv, 1)
        s.masked_fill_((torch.arange(s.shape[3], device=DEV) > last[..., None])[:, None], -math.inf)
    top = s.amax(3, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(3, keepdim=True)
    y = (p @ _pages(st, 1)) / total
    y = y.view(seqs, kv, most, h // kv, -1).transpose(1, 2).flatten(2, 3)[b, i].to(q.dtype)
    if not c["lse"]:
        return y
    lse = (top + torch.log(total)).view(seqs, kv, most, h // kv).transpose(1, 2).flatten(2, 3)[b, i]
    return [y, lse]


def _importance_plain(st):
    s = _scores(st["q"][:, None], st)
    if st["case"]["lse"]:
        p = torch.exp(s - st["lse"].view(*s.shape[:3], 1))
    else:
        p = torch.exp(s - s.amax(3, keepdim=True))
        p = p / p.sum(3, keepdim=True)
    return p.mean((1, 2))[:, :st["most"]].contiguous()


# ----------------------------------------------------------------------- run
def _cache(st):
    if "handle" not in st:
        st["handle"] = _ops().Fp8KVCache.wrap(*st["cache"])
    return st["handle"]


def run(state):
    c = state["case"]
    kind = c["kind"]
    if kind == "rotate":
        if own:
            if "sections" not in state:
                state["sections"] = [int(v) for v in c["sections"].split(",")]
            return list(_ops().rotate_positions(
                state["q"], state["k"], state["positions"], state["inv"], state["sections"],
                interleaved=c["interleaved"], adjacent=c["adjacent"], inverse=c["inverse"]))
        return [_rotate_plain(state["q"], state, c), _rotate_plain(state["k"], state, c)]
    if kind == "append":
        if own:
            cache = _cache(state)
            cache.append(state["k"], state["v"], state["table"], state["lengths"], state["starts"])
            return [cache.k, cache.v, cache.k_scale, cache.v_scale]
        k, v, ks, vs = state["cache"]
        _append_plain(state["k"], k, ks, _pack_k, _unpack_k, state)
        _append_plain(state["v"], v, vs, _pack_v, _unpack_v, state)
        return [k, v, ks, vs]
    if kind == "attend":
        if own:
            y = _cache(state).attend(state["q"], state["table"], state["lengths"], state["starts"], causal=c["causal"],
                                     return_lse=c["lse"])
            return list(y) if c["lse"] else y
        return _attend_plain(state["q"], state)
    if own:
        return _cache(state).importance(state["q"], state["table"], state["lengths"], lse=state.get("lse"),
                                        out_len=state["most"])
    return _importance_plain(state)


# ------------------------------------------------------------- what is needed
def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "rotate":
        values = case["n"] * (case["heads"] + case["kv"]) * case["dim"]
        axes = case["sections"].count(",") + 1
        return {"bytes": 2 * values * size + 8 * axes * case["n"] + 2 * case["turned"], "flops": 3 * values}
    lens, new = _lens(case)
    pages = sum(-(-n // case["page"]) for n in lens)
    h, kv, d, dv = case["heads"], case["kv"], case["dim"], case["vdim"]
    if kind == "append":
        values = sum(new) * kv * (d + dv)
        return {"bytes": values * (size + 1), "flops": 2 * values}
    if kind == "importance":
        return {"bytes": sum(lens) * kv * d + 4 * pages * (1 + kv) + sum(new) * h * d * size
                + 4 * case["seqs"] * max(lens) + (4 * case["seqs"] * h if case["lse"] else 0),
                "flops": 2 * sum(lens) * h * d}
    seen = sum(n * (ln - n) + (n * (n + 1) // 2 if case["causal"] else n * n) for ln, n in zip(lens, new))
    return {"bytes": sum(lens) * kv * (d + dv) + 4 * pages * (1 + 2 * kv) + sum(new) * h * (d + dv) * size
            + (4 * sum(new) * h if case["lse"] else 0), "flops": 2 * seen * h * (d + dv)}


# ------------------------------------------------------- the definition, in 64 bits
def _rotate_64(x, st, c):
    y = x.double().clone()
    half = c["turned"] // 2
    sections = [int(v) for v in c["sections"].split(",")]
    for i in range(half):
        if c["interleaved"]:
            a = i % len(sections)
            a = a if i < len(sections) * sections[a] else 0
        else:
            a = next(k for k in range(len(sections)) if i < sum(sections[:k + 1]))
        angle = st["positions"][a].double() * float(st["inv"][i]) * (-1.0 if c["inverse"] else 1.0)
        lo, hi = (2 * i, 2 * i + 1) if c["adjacent"] else (i, half + i)
        z = torch.complex(x[..., lo].double(), x[..., hi].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[..., lo], y[..., hi] = z.real, z.imag
    return y


def _cell_index(page, d, transposed):
    """Token and column of every byte of a page, [page / 32, D / 32, 64, 16] each."""
    t, j, l, e = np.meshgrid(np.arange(page // 32), np.arange(d // 32), np.arange(64), np.arange(16), indexing="ij")
    if transposed:
        token, col = 16 * (e // 8) + 8 * (e // 4 % 2) + 4 * (l // 32) + e % 4, 32 * j + l % 32
    else:
        token, col = l % 32, 32 * j + 16 * (l // 32) + e
    return torch.from_numpy(32 * t + token).to(DEV), torch.from_numpy(col).to(DEV)


def _of_sequence(t, which, b, head, n):
    """Keys or values [n, D] of one sequence and head, in 64 bits."""
    c = t["case"]
    page = c["page"]
    ids = t["table"][b, :-(-n // page)].long()
    token, col = _cell_index(page, (c["dim"], c["vdim"])[which], which == 1)
    raw = t["cache"][which][ids, head].to(torch.float32).double() * t["cache"][2 + which][ids, head].double()[:, None, None, None, None]
    out = torch.zeros(len(ids), page, (c["dim"], c["vdim"])[which], dtype=torch.float64, device=DEV)
    out[:, token, col] = raw
    return out.view(len(ids) * page, -1)[:n]


def _e4m3_64(v):
    """Nearest e4m3 value (ties to even) of |v| <= 448, in float64."""
    a = v.abs()
    e = torch.frexp(a).exponent.double() - 1.0
    step = torch.exp2(torch.clamp(e, min=-6.0) - 3.0)
    return torch.sign(v) * torch.round(a / step) * step


def _append_64(t, which, lens, new):
    c = t["case"]
    page, src = c["page"], t["v" if which else "k"].double()
    values = t["cache"][which].to(torch.float32).double()
    scale = t["cache"][2 + which].double()
    token, col = _cell_index(page, values.shape[3] * 32, which == 1)
    first = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for p in range((n - m) // page, -(-n // page)):
            lo, hi = max(n - m, p * page), min(n, (p + 1) * page)
            at = int(t["table"][b, p])
            rows = src[first + lo - (n - m):first + hi - (n - m)]  # [new, kv, D]
            top = rows.abs().amax((0, 2))
            e = torch.ceil(torch.log2(top / E4M3_MAX))
            e = torch.where(top / torch.exp2(e) > E4M3_MAX, e + 1, e)
            e = torch.where(top / torch.exp2(e - 1) <= E4M3_MAX, e - 1, e)
            s = torch.where(top > 0, torch.exp2(e), torch.ones_like(e))
            old = scale[at].clone()
            if lo > p * page:
                s = torch.maximum(s, old)
            cells = torch.zeros(c["kv"], page, values.shape[3] * 32, dtype=torch.float64, device=DEV)
            cells[:, token, col] = values[at]
            if lo > p * page:
                held = cells[:, :lo - p * page]
                cells[:, :lo - p * page] = _e4m3_64(held * (old / s)[:, None, None])
            cells[:, lo - p * page:hi - p * page] = _e4m3_64(rows.transpose(0, 1) / s[:, None, None])
            values[at], scale[at] = cells[:, token, col], s
        first += m
    return values, scale


def exact(case, seed):
    t = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotate":
        return [_rotate_64(t["q"], t, case), _rotate_64(t["k"], t, case)]
    lens, new = _lens(case)
    if kind == "append":
        (k, ks), (v, vs) = _append_64(t, 0, lens, new), _append_64(t, 1, lens, new)
        return [k, v, ks, vs]
    h, group = case["heads"], case["heads"] // case["kv"]
    q = t["q"].double()
    if kind == "importance":
        out = torch.zeros(case["seqs"], max(lens), dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            for j in range(case["kv"]):
                keys = _of_sequence(t, 0, b, j, n)
                for i in range(j * group, (j + 1) * group):
                    s = keys @ q[b, i] / math.sqrt(case["dim"])
                    p = torch.exp(s - t["lse"][b, i].double()) if case["lse"] else torch.softmax(s, 0)
                    out[b, :n] += p / h
        return out
    y = torch.zeros(q.shape[0], h, case["vdim"], dtype=torch.float64, device=DEV)
    lse = torch.zeros(q.shape[0], h, dtype=torch.float64, device=DEV)
    first = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        rows = slice(first, first + m)
        hidden = None
        if case["causal"]:
            hidden = torch.arange(n, device=DEV)[None] > (n - m + torch.arange(m, device=DEV))[:, None]
        for j in range(case["kv"]):
            keys, vals = _of_sequence(t, 0, b, j, n), _of_sequence(t, 1, b, j, n)
            for i in range(j * group, (j + 1) * group):
                s = q[rows, i] @ keys.T / math.sqrt(case["dim"])
                if hidden is not None:
                    s = s.masked_fill(hidden, -math.inf)
                y[rows, i] = torch.softmax(s, 1) @ vals
                lse[rows, i] = torch.logsumexp(s, 1)
        first += m
    return [y, lse] if case["lse"] else y

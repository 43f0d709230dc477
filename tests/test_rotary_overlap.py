"""What rotate_positions and the attention take as memory that two views share."""

import random

import pytest
import torch

from table_moe.ops.rotary import overlap, rows_apart


def elements(t):
    idx = torch.zeros(t.shape, dtype=torch.long)
    for dim, (s, m) in enumerate(zip(t.stride(), t.shape)):
        idx += (torch.arange(m) * s).view([-1 if i == dim else 1 for i in range(3)])
    return set((idx + t.storage_offset()).reshape(-1).tolist())


@pytest.mark.parametrize("n,h,d", [(7, 3, 8), (1, 3, 8), (7, 1, 8), (1, 1, 8)])
def test_columns_of_a_fused_row_do_not_overlap(n, h, d):
    """q, k and v next to each other, by turns, by turns within groups, heads before tokens."""
    f = torch.zeros(n, 3 * h, d)
    layouts = {
        "next": [f[:, i * h:(i + 1) * h] for i in range(3)],
        "turns": [f.view(n, h, 3, d)[:, :, i] for i in range(3)],
        "columns": [f.view(n, h, 3 * d)[:, :, i * d:(i + 1) * d] for i in range(3)],
        "heads first": [f.view(3, h, n, d)[i].transpose(0, 1) for i in range(3)],
        "heads first, turns": [f.view(h, 3, n, d)[:, i].transpose(0, 1) for i in range(3)],
        "heads first, columns": [f.view(h, n, 3 * d)[..., i * d:(i + 1) * d].transpose(0, 1) for i in range(3)],
    }
    for name, views in layouts.items():
        for i, x in enumerate(views):
            assert rows_apart(x), name
            for j, y in enumerate(views):
                assert overlap(x, y) == (i == j), (name, i, j)
                assert bool(elements(x) & elements(y)) == (i == j), (name, i, j)


def test_what_overlaps_is_seen():
    """Random views of one buffer: none that share an element pass for apart."""
    r = random.Random(1)
    buf = torch.zeros(4000)
    apart = shared = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            n, h, d = r.choice([1, 2, 5]), r.choice([1, 2, 3]), r.choice([1, 4, 8])
            unit = r.choice([d, 2 * d, 3 * d, 8])
            sh = unit * r.choice([1, 2, 3])
            st = r.choice([sh * h, sh * h + unit, unit * r.choice([1, 2, 5, 7])])
            v = buf.as_strided((n, h, d), (st, sh, 1), r.randint(0, 60))
            if not rows_apart(v):
                break
            views.append(v)
        if len(views) < 2:
            continue
        both = bool(elements(views[0]) & elements(views[1]))
        says = overlap(*views)
        assert says or not both, [(tuple(v.shape), v.stride(), v.storage_offset()) for v in views]
        apart, shared = apart + (not says), shared + both
    assert apart > 200 and shared > 200


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 9])
def test_rotate_in_place_by_turns(hip_device, n):
    """q, k and v of a head next to each other in a fused row: q and k are turned in place, v stays."""
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(61)
    h, d = 4, 64
    f = torch.randn(n, h, 3, d, generator=g).to(torch.bfloat16).to(dev)
    was = f.clone()
    pos, inv = torch.arange(n, device=dev) + 100, torch.rand(d // 2, generator=g).to(dev)
    q, k = f[:, :, 0], f[:, :, 1]
    want = rotate_positions(q.clone(), k.clone(), pos, inv)
    rotate_positions(q, k, pos, inv, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(f[:, :, 2], was[:, :, 2])
    g2 = was.clone()
    rotate_positions(g2[:, :, 0], g2[:, :, 1], pos, inv, out=(g2[:, :, 2], torch.empty_like(k)))
    assert torch.equal(g2[:, :, 2], want[0]) and torch.equal(g2[:, :, :2], was[:, :, :2])

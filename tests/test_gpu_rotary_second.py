"""Second-order gradients of rotate_positions against their closed form."""

import pytest
import torch

from test_gpu_kv8 import rotate_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved,adjacent,inverse", [(False, False, False), (True, False, True), (True, True, False)])
def test_second_order(hip_device, interleaved, adjacent, inverse):
    """o = R q and k' = R k: d / dq of the sum of d / dq of sum(o^3) is R^T (6 o x R 1), of sum(k'^3) likewise."""
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(81)
    n, h, kv, d, sec = 11, 3, 2, 80, (12, 10, 10)
    pos = torch.randint(0, 5000, (3, n), generator=g)
    inv = (1e4 ** (-torch.arange(32).double() / 32)).float()
    how = dict(interleaved=interleaved, adjacent=adjacent, inverse=inverse)
    ref = lambda t, back=False: rotate_ref(t, pos, inv, sec, interleaved, adjacent, inverse != back)  # noqa: E731
    xs = [torch.randn(n, m, d, generator=g) for m in (h, kv)]
    q, k = (x.to(dev).requires_grad_() for x in xs)
    y, z = rotate_positions(q, k, pos.to(dev), inv.to(dev), sec, **how)
    first = torch.autograd.grad((y ** 3).sum() + (z ** 3).sum(), (q, k), create_graph=True)
    second = torch.autograd.grad(first[0].sum() + first[1].sum(), (q, k))
    for x, got in zip(xs, second):
        o, so = ref(x)
        w, sw = ref(torch.ones_like(x))
        t = 6 * o * w
        want, st = ref(t, True)
        # a rotation is off by 6e-7 of the pair's sizes (columns that are not turned: not at all, their sizes are 0 here),
        # each of four products by 2^-24; then the pair of errors is turned, and the result off as any rotation
        et = 6 * (6e-7 * so * w.abs() + o.abs() * 6e-7 * sw + 4 * 2.0 ** -24 * (o * w).abs())
        turned = ref(et, True)[1]
        tol = torch.where(st > 0, turned + 6e-7 * st, et)
        assert bool(((got.cpu().double() - want).abs() <= tol * 1.01 + 1e-12).all())

"""Forward-mode derivatives of rotate_positions."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_kv8 import BF16, F16, F32, rotate_close, rotate_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved,adjacent,inverse", [(True, False, False), (False, True, True)])
def test_tangents(hip_device, dt, interleaved, adjacent, inverse):
    from table_moe.ops import rotate_positions

    dev = hip_device
    g = torch.Generator().manual_seed(51)
    n, h, kv, d, sec = 9, 4, 2, 96, (10, 12, 10)
    pos = torch.randint(0, 90000, (3, n), generator=g)
    inv = (1e5 ** (-torch.arange(32).double() / 32)).float()
    q, k, tq, tk = (torch.randn(n, x, d, generator=g).to(dt) for x in (h, kv, h, kv))
    how = dict(interleaved=interleaved, adjacent=adjacent, inverse=inverse)
    args = (pos.to(dev), inv.to(dev), sec)
    plain = rotate_positions(q.to(dev), k.to(dev), *args, **how)
    with fwd.dual_level():
        y, z = rotate_positions(fwd.make_dual(q.to(dev), tq.to(dev)), fwd.make_dual(k.to(dev), tk.to(dev)), *args, **how)
        for out, p, t in ((y, plain[0], tq), (z, plain[1], tk)):
            primal, tangent = fwd.unpack_dual(out)
            assert torch.equal(primal, p)
            rotate_close(tangent, *rotate_ref(t, pos, inv, sec, interleaved, adjacent, inverse), 64)
        y, _ = rotate_positions(fwd.make_dual(q.to(dev), tq.to(dev)), None, *args, **how)
        rotate_close(fwd.unpack_dual(y).tangent, *rotate_ref(tq, pos, inv, sec, interleaved, adjacent, inverse), 64)

"""rotate_positions in place on a single token or head, whose strides mean nothing."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,h", [(1, 4), (5, 1), (1, 1)])
def test_in_place_whatever_the_stride_of_one(hip_device, n, h):
    from table_moe.ops import rotate_positions

    dev, d = hip_device, 64
    g = torch.Generator().manual_seed(71)
    x = torch.randn(n, h, d, generator=g).to(torch.float16).to(dev)
    pos, inv = torch.arange(n, device=dev) + 9, torch.rand(d // 2, generator=g).to(dev)
    want, _ = rotate_positions(x, None, pos, inv)
    st, sh = x.stride()[:2]
    view = x.as_strided(x.shape, (7 if n == 1 else st, 13 if h == 1 else sh, 1))  # the same elements
    for q, out in ((x.clone(), None), (x, view)):
        if out is None:
            out = q.as_strided(q.shape, view.stride())
        got, _ = rotate_positions(q, None, pos, inv, out=(out, None))
        assert got is out and torch.equal(q, want)
    with pytest.raises(ValueError, match="overlap"):  # two columns on: other elements of the same memory
        wide = torch.zeros(n * h * d + 8, dtype=torch.float16, device=dev)
        rotate_positions(wide[:n * h * d].view(n, h, d), None, pos, inv, out=(wide[2:2 + n * h * d].view(n, h, d), None))

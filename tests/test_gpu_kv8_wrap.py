"""Fp8KVCache.wrap: which scales it takes."""

import math

import pytest
import torch

BAD = [1.5, 3.0, -1.0, -0.0, 2.0 ** -101, 2.0 ** 121, math.nan, math.inf, 1e-45, 0.0078]


def test_scales_on_the_host():
    from table_moe.ops.fp8_cache import _scales_hold

    good = torch.tensor([2.0 ** e for e in range(-100, 121)] + [0.0])
    assert _scales_hold(good) and _scales_hold(good[:0])
    for x in BAD:
        assert not _scales_hold(torch.cat([good, torch.tensor([x])])), x


@pytest.mark.gpu
def test_wrap_refuses_other_scales(hip_device):
    """A value's scale with a mantissa lost it (values up to twice too small), without an error."""
    from table_moe.ops import Fp8KVCache

    dev = hip_device
    g = torch.Generator().manual_seed(2)
    c = Fp8KVCache(5, 3, 64, page_size=32, device=dev)
    k = torch.randn(100, 3, 64, generator=g).to(dev)
    table, lengths = torch.arange(4, dtype=torch.int32, device=dev)[None], torch.tensor([100], device=dev)
    c.append(k, k, table, lengths, torch.tensor([0, 100], device=dev))
    w = Fp8KVCache.wrap(c.k, c.v, c.k_scale, c.v_scale)
    q = torch.randn(1, 6, 64, generator=g).to(torch.float16).to(dev)
    assert torch.equal(w.attend(q, table, lengths), c.attend(q, table, lengths))
    for x in BAD:
        for i in (0, 1):
            s = [c.k_scale.clone(), c.v_scale.clone()]
            s[i][3, 2] = x
            with pytest.raises(ValueError, match="scales"):
                Fp8KVCache.wrap(c.k, c.v, *s)
    # storage that nobody has written to: zeros
    z = Fp8KVCache.wrap(torch.zeros_like(c.k.view(torch.uint8)).view(c.k.dtype), torch.zeros_like(c.v.view(torch.uint8)).view(c.v.dtype),
                        torch.zeros_like(c.k_scale), torch.zeros_like(c.v_scale))
    z.append(k, k, table, lengths, torch.tensor([0, 100], device=dev))
    assert torch.equal(z.attend(q, table, lengths), c.attend(q, table, lengths))


@pytest.mark.gpu
def test_wrap_while_capturing(hip_device):
    from table_moe.ops import Fp8KVCache

    dev = hip_device
    c = Fp8KVCache(2, 1, 64, page_size=32, device=dev)
    g = torch.Generator().manual_seed(4)
    k = torch.randn(40, 1, 64, generator=g).to(dev)
    table, lengths = torch.arange(2, dtype=torch.int32, device=dev)[None], torch.tensor([40], dtype=torch.int32, device=dev)
    c.append(k, k, table, lengths, torch.tensor([0, 40], device=dev))
    q = torch.randn(1, 2, 64, generator=g).to(torch.bfloat16).to(dev)
    want = c.attend(q, table, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attend(q, table, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = Fp8KVCache.wrap(c.k, c.v, c.k_scale, c.v_scale).attend(q, table, lengths)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(c.attend(q, table, lengths), want)

"""64-bit tables, lengths and starts of the 8-bit cache whose entries 32 bits do not hold."""

import pytest
import torch

from test_gpu_kv8 import BF16, filled

gpu = pytest.mark.gpu

FAR = 2 ** 32


@pytest.fixture
def batch(hip_device):
    g = torch.Generator().manual_seed(3)
    cache, _ = filled(g, 6, 2, 32, 64, 64, hip_device)
    mk = lambda n, h: torch.randn(n, h, 64, generator=g).to(BF16).to(hip_device)  # noqa: E731
    return cache, mk


def held(cache):
    return [t.view(torch.uint8).clone() for t in (cache.k, cache.v)] + [cache.k_scale.clone(), cache.v_scale.clone()]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_int32_conversion_keeps_what_is_out_of_range():
    """(of the helper itself, on the host's tensors)"""
    from table_moe.ops.fp8_cache import _int32

    t = torch.tensor([5, FAR + 5, -FAR + 5, 2 ** 31, -1, 2 ** 63 - 1, -2 ** 63])
    assert _int32("lengths", t, 1).tolist() == [5, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -1, 2 ** 31 - 1, -2 ** 31]


@gpu
@pytest.mark.parametrize("entry", [FAR + 2, -FAR + 2, 2 ** 63 - 1, 2 ** 31, 2 ** 33 + 5])
def test_page_numbers(batch, hip_device, entry):
    """A page number past 32 bits is a page that is not there, not the one of its low bits."""
    cache, mk = batch
    dev = hip_device
    far = torch.tensor([[0, entry], [4, 5]], device=dev)
    none = torch.tensor([[0, -1], [4, 5]], dtype=torch.int32, device=dev)
    lengths, starts = torch.tensor([50, 60], device=dev), torch.tensor([0, 40, 45], device=dev)
    before = held(cache)
    k, v = mk(45, 2), mk(45, 2)
    cache.append(k, v, none, lengths, starts)
    want = held(cache)
    for t, x in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), before):
        t.copy_(x)
    cache.append(k, v, far, lengths, starts)
    assert same(held(cache), want)
    q = mk(2, 4)
    a, b = cache.attend(q, far, lengths, return_lse=True), cache.attend(q, none, lengths, return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(cache.importance(q, far, lengths), cache.importance(q, none, lengths))


@gpu
def test_lengths_and_starts(batch, hip_device):
    """A length of 2^32 + 3 ends with the table as any other past it; one of -2^32 + 3 is none; starts of 2^32 are past the rows."""
    cache, mk = batch
    dev = hip_device
    table = torch.tensor([[0, 1], [2, 3]], device=dev)
    q = mk(2, 4)
    for far, near in ((FAR + 3, 64), (2 ** 31, 64), (-FAR + 3, 0)):
        x, y = torch.tensor([far, 20], device=dev), torch.tensor([near, 20], device=dev)
        assert torch.equal(cache.attend(q, table, x), cache.attend(q, table, y))
        assert torch.equal(cache.importance(q, table, x), cache.importance(q, table, y))
    q, out = mk(8, 4), torch.full((8, 4, 64), 7.0, dtype=BF16, device=dev)
    lengths = torch.tensor([30, 20], device=dev)
    want = cache.attend(q, table, lengths, torch.tensor([0, 8, 8], device=dev))
    cache.attend(q, table, lengths, torch.tensor([0, FAR + 3, FAR + 3], device=dev), out=out)
    assert torch.equal(out, want)
    before = held(cache)
    cache.append(mk(8, 2), mk(8, 2), table, torch.tensor([-FAR + 30, FAR + 64], device=dev), torch.tensor([0, 8, 8], device=dev))
    assert same(held(cache), before)

"""The tensors of an Fp8KVCache, whose addresses its calls use, cannot be exchanged (on the host, with the check for a
device replaced)."""

import ctypes as C
import gc
import weakref

import pytest
import torch

from table_moe.ops import fp8_cache


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(fp8_cache.N, "require_hip", lambda *t: torch.device("cpu"))
    return fp8_cache.Fp8KVCache(3, 2, 64, page_size=32, device="cpu")


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_tensors_are_not_assigned(cache, name):
    t = getattr(cache, name)
    with pytest.raises(AttributeError):
        setattr(cache, name, t.clone())
    with pytest.raises(AttributeError):
        delattr(cache, name)
    assert getattr(cache, name) is t and getattr(cache._desc, name) == t.data_ptr()


def test_tensors_live_as_long_as_the_cache(cache):
    refs = [weakref.ref(getattr(cache, n)) for n in ("k", "v", "k_scale", "v_scale")]
    gc.collect()
    assert all(r() is not None for r in refs)
    cache.k_scale.fill_(2.0)  # in place, which is what a user does
    at = (C.c_float * 6).from_address(cache._desc.k_scale)
    assert list(at) == [2.0] * 6

"""Evictions whose target cache has been closed; no device needed."""
import types

import pytest
import torch

from gufo_npu_b200 import _capi
from gufo_npu_b200.cache8 import CudaCache8


def cache(ctx, handle):
    c = object.__new__(CudaCache8)
    c.ctx, c.handle, c.kv_heads = ctx, handle, 2
    return c


def test_evict_into_a_closed_cache_is_refused(monkeypatch):
    """A closed cache's handle is 0, which the library takes for an eviction in place: the source would lose its rows."""
    calls = []
    monkeypatch.setattr(_capi, "native", types.SimpleNamespace(cache8_evict=lambda *args: calls.append(args) or 0))
    ctx = types.SimpleNamespace(device=0, _address=1, _check=lambda status: None)
    batch = types.SimpleNamespace(device=0, sequences=1, args=None)
    kept = torch.zeros(1, 2, 8, dtype=torch.int32)
    source = cache(ctx, 5)
    for slots in (None, [0]):
        with pytest.raises(ValueError, match="closed"):
            source.evict_device(batch, 8, kept, into=cache(ctx, 0), into_slots=slots)
    assert not calls
    source.evict_device(batch, 8, kept, into=cache(ctx, 7))
    source.evict_device(batch, 8, kept)
    assert [args[-2] for args in calls] == [7, 0]

"""CPU: the bookkeeping of a layer's cache, the kernels stubbed."""

import pytest
import torch

from lockstep_amd import fp4_attention as A


def _cache(**kw):
    return A.LayerCache(3, 40, 2, 64, page_size=16, track=True, device="cpu", **kw)


def test_evict_keeps_the_tensors(monkeypatch):
    """A captured step reads and writes lengths, table and weights where they were."""
    c = _cache()
    lengths, table, other, weights = c.lengths, c.table, c.other, c.weights
    first, second = table.clone(), other.clone()
    kept = torch.rand(3, 2, 20)

    def evict(pages, t, n, w, keep, out, **kw):
        assert torch.equal(t, first) and torch.equal(out, second)
        return torch.zeros(3, 2, keep), kept, torch.tensor([20, 7, 0], dtype=torch.int32)
    monkeypatch.setattr(A.kv_cache, "evict", evict)
    c.grow(30, torch.tensor([30, 7, 0], dtype=torch.int32))
    c.evict(20)
    assert c.lengths is lengths and c.table is table and c.other is other and c.weights is weights
    assert lengths.tolist() == [20, 7, 0] and c.used == 20
    assert torch.equal(table, second) and torch.equal(other, first)
    assert torch.equal(weights[:, :, :20], kept) and (weights[:, :, 20:] == 0).all()


def test_reserve_counts_what_a_replay_adds():
    c = _cache()
    c.grow(10, 10)
    c.reserve(30)
    assert c.used == 40 and c.lengths.tolist() == [10, 10, 10]
    with pytest.raises(ValueError, match="holds 40"):
        c.reserve(1)
    assert c.used == 40

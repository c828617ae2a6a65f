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


@pytest.fixture
def layer(monkeypatch):
    """A layer whose linears give zeros and whose attention is not reached."""
    l = A.MXFP4SelfAttention(256, 4, 2).to(torch.bfloat16)
    l.packed = ((512, None), (256, None))
    monkeypatch.setattr(A, "mxfp4_linear_w", lambda x, n, s: x.new_zeros((*x.shape[:-1], n)))
    return l


def test_refused_calls_leave_the_cache_as_it_was(layer):
    """Wrong batches, offsets and types are errors; no token of theirs is counted."""
    c = layer.new_cache(3, 40, page_size=16, track=True)
    x, off = torch.zeros((7, 256)).bfloat16(), torch.tensor([0, 3, 5, 7], dtype=torch.int32)
    calls = [lambda: layer.prefill(x, c, off[:3]),            # two prompts for three sequences
             lambda: layer.prefill(x, c, off.cpu()),          # CPU tensors
             lambda: layer.step(torch.zeros((2, 1, 256)).bfloat16(), c),
             lambda: layer.step(torch.zeros((3, 1, 256)), c),
             lambda: c.grow(1, torch.zeros(2, dtype=torch.int32))]
    for call in calls:
        with pytest.raises((ValueError, AssertionError, TypeError, RuntimeError)):
            call()
        assert c.used == 0 and c.lengths.tolist() == [0, 0, 0]


def test_prompt_weights_stay_within_the_rows(layer, monkeypatch):
    """Offsets past the rows, or before them, are cut to them, as the kernels cut them."""
    seen = []

    def attend(q, pages, table, lengths, **kw):
        seen.append(q.shape)
    monkeypatch.setattr(A.kv_cache, "attend", attend)
    c = _cache()
    for off, longest in (([0, 3, 5, 900], 7), ([0, 3, 2 ** 31 - 1, 7], 40), ([-5, -3, 5, 7], 7), ([0, 3, 5, 7], 0)):
        layer._prompt_weights(torch.zeros((7, 4, 64)), c, torch.tensor(off, dtype=torch.int32), longest)
    assert seen == [(3, 7, 4, 64), (3, 40, 4, 64), (3, 7, 4, 64)]


@pytest.mark.parametrize("batch,tokens", [(0, 40), (2, 0)])
def test_an_empty_cache(batch, tokens):
    for track in (True, False):
        c = A.LayerCache(batch, tokens, 2, 64, page_size=16, track=track, device="cpu")
        assert c.table.shape == c.other.shape == (batch, -(-tokens // 16)) and c.lengths.shape == (batch,)

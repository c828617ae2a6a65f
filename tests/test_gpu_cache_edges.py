"""The cache's operators at their edges: tables with ids outside the pool, inputs
whose axes of one element have odd strides."""

import pytest
import torch

from .test_gpu_kv_cache import filled, formula, held, reference_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,page,keep,sinks,recent,gone", [
    ([300], 16, 100, 4, 30, (0, 3, 18)),             # among the sinks, the candidates, the last
    ([300, 90], 16, 260, 0, 0, (1, 2, 5)),           # more stay than are there
    ([300, 40], 16, 64, 2, 8, (1, 4)),
    ([5000], 64, 700, 0, 100, (0, 20, 21, 78)),      # 8 positions a thread
    ([33000], 1024, 9000, 3, 10, (1, 31)),           # read again in each round
    ([64], 64, 10, 1, 1, (0,)),                      # none is left
])
def test_evict_leaves_out_what_is_in_no_page(lens, page, keep, sinks, recent, gone, dev):
    """Tokens of an id outside the pool are hidden: they do not stay, and are not
    counted, and nothing that lay in the new pages comes in their place."""
    from lockstep_amd import kv_cache as kc
    Hkv, D, B = 2, 64, len(lens)
    pages, table, lengths, _, _ = filled(lens, Hkv, D, page, torch.bfloat16, dev, seed=keep)
    cap, n0, spare = table.shape[1] * page, pages[0].shape[0], -(-keep // page)
    g = torch.Generator(device=dev).manual_seed(keep)
    grown = kc.Pages(*(torch.cat([t, torch.randint(0, 255, (B * spare, *t.shape[1:]), generator=g, device=dev).to(t.dtype)])
                       for t in pages))
    for i, p in enumerate(gone):
        table[0, p] = -1 if i % 2 else n0 + B * spare
    out_table = (torch.randperm(B * spare).to(torch.int32) + n0).reshape(B, spare).to(dev)
    w = torch.randint(0, 9, (B, Hkv, cap), generator=g, device=dev).float()
    index, kept, new = kc.evict(grown, table, lengths, w, keep, out_table, sinks=sinks, recent=recent)
    safe = table.clamp(0, n0 - 1)
    q = torch.randn((B, 1, 4, D), generator=g, device=dev).bfloat16()
    o = kc.attend(q, grown, out_table, new)
    for b, n in enumerate(lens):
        there = [j for j in range(n) if b or j // page not in gone]
        c0, c1 = min(sinks, n), max(min(sinks, n), n - recent)
        for h in range(Hkv):
            # the protected are those by position; of the others in their order the largest
            free = [j for j in there if c0 <= j < c1]
            fixed = [j for j in there if not c0 <= j < c1]
            wl = w[b, h].tolist()
            best = [free[i] for i in reference_evict([wl[j] for j in free], len(free), max(0, keep - len(fixed)), 0, 0)] \
                if keep > len(fixed) else []
            want = sorted(fixed + best)
            m = len(want)
            assert m == min(len(there), keep) == new[b].item()
            assert index[b, h].tolist() == want + [-1] * (keep - m)
            at = torch.tensor(want, device=dev, dtype=torch.long)
            assert torch.equal(kept[b, h, :m], w[b, h, at]) and (kept[b, h, m:] == 0).all()
            for s, d in zip(held(grown, safe, b, n, page, dev), held(grown, out_table, b, m, page, dev)):
                assert torch.equal(s[at, h], d[:, h])
        if not there:
            assert (o[b] == 0).all()


def test_append_of_one_token_with_an_odd_stride(dev):
    """The stride of an axis of one element means nothing."""
    from lockstep_amd import fp4
    from lockstep_amd import kv_cache as kc
    base = torch.randn((3, 513), device=dev).half()
    x = base[:, :512].view(3, 1, 8, 64)[0:1]
    assert x.stride(0) % 8 and x.data_ptr() % 16 == 0
    pages = kc.new_pages(1, 8, 64, 16, device=dev)
    table, lengths = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    kc.append(pages, x, x, table, lengths)
    codes, scale = fp4.quantize_pack_mxfp4(x[0, 0].contiguous())
    for c, s in (pages[:2], pages[2:]):
        assert torch.equal(c[0, :, 0], codes) and torch.equal(s[0, :, 0], scale)


@pytest.mark.parametrize("values", [1, "yes", True])
def test_append_returns_values_for_any_true_flag(values, dev):
    from lockstep_amd import kv_cache as kc
    pages = kc.new_pages(1, 2, 64, 16, device=dev)
    table, lengths = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.full((1,), 3, dtype=torch.int32, device=dev)
    x = torch.randn((1, 3, 2, 64), device=dev).bfloat16()
    k, v = kc.append(pages, x, x, table, lengths, values=values)
    assert torch.equal(k, v) and k.shape == x.shape
    assert kc.append(pages, x, x, table, lengths, values=0) is None

"""A paged key-value cache in MXFP4, and the operators of serving from it.

The cache holds keys and values in the format of the framework's weights and
activations (fp4.quantize_pack_mxfp4: E2M1 codes, one E8M0 scale per 32
elements along the head), 17 bytes per 32 elements against 64 in bf16.  It is
a pool of pages that sequences own through a block table:

    pages = new_pages(n, kv_heads, head_dim, page_size)
    lengths += new                                  # device int32 [B]
    append(pages, k, v, table, lengths)             # quantize into the pages
    o = attend(q, pages, table, lengths, window=..., sinks=..., weights=w)
    index, w, lengths = evict(pages, table, lengths, w, keep, out_table)

table is int32 [B, max_pages] and lengths int32 [B], both on the device; token
j of sequence b lies in page table[b, j // page], slot j % page.  Entries past
a sequence's pages are never read.  No call synchronizes, or is differentiable.  Kernels:
lockstep_amd/csrc/kv_cache.hip, and attention.hip for many rows.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _capi as C
from .attention import _strides, check_mask, rows16


class Pages(NamedTuple):
    """The pool: uint8 [pages, kv_heads, page, D // 2] codes and
    [pages, kv_heads, page, D // 32] E8M0 scales, of keys and of values."""
    k_codes: torch.Tensor
    k_scale: torch.Tensor
    v_codes: torch.Tensor
    v_scale: torch.Tensor


def new_pages(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> Pages:
    """An empty pool.  page_size: a power of two, 16 to 1024; head_dim 64 or 128."""
    _check_format(head_dim, page_size)
    one = lambda n: torch.zeros((pages, kv_heads, page_size, n), dtype=torch.uint8, device=device)  # noqa: E731
    return Pages(one(head_dim // 2), one(head_dim // 32), one(head_dim // 2), one(head_dim // 32))


def _check_format(D, page):
    assert D in (64, 128), f"head_dim={D} must be 64 or 128"
    assert 16 <= page <= 1024 and page & (page - 1) == 0, f"page={page} must be a power of two, 16 to 1024"


def _cache(pages, table, lengths):
    """The C description of a cache; the tensors are checked first."""
    kc, ks, vc, vs = pages
    C.require_device(kc, ks, vc, vs, table, lengths)
    assert kc.dim() == 4 and kc.shape == vc.shape, "codes must be [pages, kv_heads, page, D // 2]"
    n, h, page, half = kc.shape
    D = 2 * half
    _check_format(D, page)
    assert ks.shape == vs.shape == (n, h, page, D // 32), "scales must be [pages, kv_heads, page, D // 32]"
    for t in (kc, ks, vc, vs):
        assert t.dtype == torch.uint8 and t.is_contiguous(), "the pool's tensors are contiguous uint8"
    assert h > 0, "no key heads"
    assert table.dim() == 2 and table.dtype == torch.int32 and table.is_contiguous(), \
        "table must be contiguous int32 [B, max_pages]"
    assert lengths.shape == table.shape[:1] and lengths.dtype == torch.int32 and lengths.is_contiguous(), \
        "lengths must be contiguous int32 [B]"
    _one_device(kc, ks, vc, vs, table, lengths)
    return C.KVCache(kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), n, page, h, D, table.data_ptr(),
                     lengths.data_ptr(), table.shape[0], table.shape[1])


def _one_device(*tensors):
    assert len({t.device for t in tensors}) == 1, "all tensors must be on one device"


def append(pages, k, v, table, lengths, *, offsets=None, values=False):
    """Quantize new tokens' keys and values into the cache.

    k, v [B, T, Hkv, D] (bf16 or fp16, any strides): the T newest tokens of
    every sequence, or with offsets (int32 [B+1]) packed [N, Hkv, D],
    sequence b's being offsets[b] .. offsets[b+1]-1.  lengths already counts
    them: they become positions lengths[b] - n_b .. lengths[b] - 1.
    Positions below 0 (padding in front) or past the table are not written.
    The bytes are those of fp4.quantize_pack_mxfp4 on each head's vector.
    With values=True returns (k, v) as now held: bf16, exact."""
    if (r := C.fast.kv_append(pages, k, v, table, lengths, offsets, values)) is not None:
        return r if values else None
    C.not_traced("append")
    c = _cache(pages, table, lengths)
    if k.dtype not in (torch.bfloat16, torch.float16) or v.dtype != k.dtype:
        raise TypeError(f"k and v must share bfloat16 or float16, got {k.dtype}, {v.dtype}")
    C.require_device(k, v)
    assert k.shape == v.shape and k.shape[-2:] == (c.kv_heads, c.head_dim), \
        f"k and v must be [.., {c.kv_heads}, {c.head_dim}], got {list(k.shape)}, {list(v.shape)}"
    if offsets is None:
        assert k.dim() == 4 and k.shape[0] == c.batch, "k and v must be [B, T, Hkv, D]"
        per = k.shape[1]
        k2, v2 = k.reshape(-1, *k.shape[2:]), v.reshape(-1, *v.shape[2:])
    else:
        assert k.dim() == 3, "with offsets, k and v must be [N, Hkv, D]"
        C.require_device(offsets)
        assert offsets.dtype == torch.int32 and offsets.shape == (c.batch + 1,) and offsets.is_contiguous(), \
            "offsets must be contiguous int32 [B + 1]"
        _one_device(offsets, table)
        per, k2, v2 = 0, k, v
    _one_device(k, v, table)
    k2, v2 = rows16(k2), rows16(v2)
    out = (torch.empty(k.shape, dtype=torch.bfloat16, device=k.device),
           torch.empty(k.shape, dtype=torch.bfloat16, device=k.device)) if values else None
    if k2.numel():
        sk, sv = _strides(k2), _strides(v2)
        C.call("lsmx_kv_append", ctypes.addressof(c), k2.data_ptr(), ctypes.addressof(sk) + 8, v2.data_ptr(),
               ctypes.addressof(sv) + 8, C.dtype_code(k.dtype), k2.shape[0], per,
               None if offsets is None else offsets.data_ptr(), out[0].data_ptr() if out else None,
               out[1].data_ptr() if out else None, C.stream_of(k))
    return out


def attend(q, pages, table, lengths, *, window=None, sinks=0, scale=None, weights=None):
    """Attention of the newest tokens over the cache.

    q [B, T, H, D] (bf16 or fp16, any strides; H a multiple of Hkv): query i of
    sequence b has position lengths[b] - T + i and sees key j when j <= its
    position and (window is None, or j > position - window, or j < sinks).
    A row that sees nothing gives 0.  Returns o [B, T, H, D] in q's type.
    Scores, softmax and sums are fp32; cached values enter as they are held
    (fp16 rows over blocks that fp16 does not hold take a slow path in fp32);
    probabilities are rounded to q's type for the product with them.

    weights (fp32 [B, Hkv, >= max_pages * page], contiguous): the softmax
    weight of every key, summed over the T tokens and the heads that share its
    head, is added in place.  Deterministic.  The result has no gradient."""
    if (r := C.fast.kv_attend(q, pages, table, lengths, window, sinks, scale, weights)) is not None:
        return r
    C.not_traced("attend")
    c = _cache(pages, table, lengths)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    C.require_device(q)
    B, T, H, D = q.shape
    assert B == c.batch and D == c.head_dim and H > 0 and H % c.kv_heads == 0, \
        f"q must be [{c.batch}, T, a multiple of {c.kv_heads}, {c.head_dim}], got {list(q.shape)}"
    _one_device(q, table)
    window, sinks, scale = check_mask(window, sinks, scale, D)
    if weights is not None:
        C.require_device(weights)
        _one_device(weights, table)
        _check_weights(weights, c)
    q = rows16(q)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if q.numel():
        n = C.load().lsmx_kv_attend_workspace(ctypes.addressof(c), T, H, window, sinks, int(weights is not None))
        ws = C.workspace(q.device, n) if n else None
        st = _strides(q)
        C.call("lsmx_kv_attend", ctypes.addressof(c), q.data_ptr(), ctypes.addressof(st), C.dtype_code(q.dtype), T, H,
               window, sinks, scale, o.data_ptr(), weights.data_ptr() if weights is not None else None,
               weights.shape[2] if weights is not None else 0, ws.data_ptr() if n else None, n, C.stream_of(q))
    return o


def _check_weights(w, c):
    cap = c.max_pages * c.page
    assert w.dtype == torch.float32 and w.is_contiguous() and w.dim() == 3 and \
        w.shape[:2] == (c.batch, c.kv_heads) and w.shape[2] >= cap, \
        f"weights must be contiguous fp32 [{c.batch}, {c.kv_heads}, at least {cap}]"


def evict(pages, table, lengths, weights, keep, out_table, *, sinks=0, recent=0):
    """Cut every sequence to its `keep` most attended tokens, head by head.

    The first `sinks` and the last `recent` tokens stay; of the others those
    with the largest weights (fp32 [B, Hkv, >= max_pages * page], as attend
    accumulates them; ties: the earlier token; a NaN counts as the largest).
    Tokens in no page (an id outside the pool) do not stay, nor count.
    What stays keeps its order and is copied to positions 0, 1, .. of the
    pages of out_table (int32 [B, pages for `keep` tokens], same pool, other
    pages than table's: the old ones are free afterwards, or still another
    sequence's).  sinks + recent <= keep.

    Returns (index int32 [B, Hkv, keep]: the positions they had, -1 past the
    last; weights fp32 [B, Hkv, keep]: theirs, 0 past the last; lengths int32
    [B]).  Afterwards positions, windows and sinks count the kept tokens."""
    if (r := C.fast.kv_evict(pages, table, lengths, weights, keep, out_table, sinks, recent)) is not None:
        return r
    C.not_traced("evict")
    c = _cache(pages, table, lengths)
    C.require_device(weights, out_table)
    _check_weights(weights, c)
    if not 1 <= keep < 2 ** 30 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"evict needs keep >= 1 and sinks + recent <= keep, got {keep}, {sinks}, {recent}")
    most = min(keep, c.max_pages * c.page)
    assert out_table.dim() == 2 and out_table.shape[0] == c.batch and out_table.dtype == torch.int32 and \
        out_table.is_contiguous() and out_table.shape[1] * c.page >= most, \
        f"out_table must be contiguous int32 [{c.batch}, pages of {c.page} for {most} tokens]"
    _one_device(weights, out_table, table)
    index = torch.empty((c.batch, c.kv_heads, keep), dtype=torch.int32, device=table.device)
    kept = torch.empty((c.batch, c.kv_heads, keep), dtype=torch.float32, device=table.device)
    new = torch.empty_like(lengths)
    if c.batch:
        C.call("lsmx_kv_evict", ctypes.addressof(c), weights.data_ptr(), weights.shape[2], keep, sinks, recent,
               out_table.data_ptr(), out_table.shape[1], index.data_ptr(), kept.data_ptr(), new.data_ptr(),
               C.stream_of(table))
    return index, kept, new

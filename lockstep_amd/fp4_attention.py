"""A self-attention layer in MXFP4, from training to serving.

What stands between the linears of a block is the reference's
train.py:46-52 with its linears replaced (fp4_linear.py:48-58); here the whole
layer runs on this package's kernels:

    layer = MXFP4SelfAttention(1024, heads=16, kv_heads=4, window=1024, sinks=4).cuda().bfloat16()
    layer(x).sum().backward()                      # x bf16; MXFP4 linears, sink_window_attention

    layer.pack()                                   # weights to MXFP4, once
    cache = layer.new_cache(batch=8, tokens=4096, track=True)
    y = layer.prefill(prompts, cache, offsets)     # packed prompts: attention over their own keys
    y = layer.step(x, cache)                       # the next tokens, over the 4-bit cache
    cache.evict(keep=2048, recent=256)             # drop the least attended
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import kv_cache
from .attention import check_mask, sink_window_attention
from .fp4 import quantize_pack_mxfp4
from .fp4_linear import MXFP4Linear
from .mxfp4_gemm import mxfp4_linear_w


_WEIGHT_ROWS = 16384  # rows of a pass over a prompt's weights (prefill)


class LayerCache:
    """One layer's MXFP4 cache: `batch` sequences of up to `tokens` tokens.

    track=True accumulates the tokens' softmax weights, of prompts and of steps,
    and holds a second set of pages for evict to move to.  lengths counts on the
    device; `used` is the host's bound on the longest of them, so that no call
    synchronizes.

    All tensors stay where they are, so that a step captured in a graph goes on
    after evictions.  Its replays count on the device alone: reserve() their tokens,
    or those past the table are dropped.  (The capture runs nothing, but is
    counted in `used`.)"""

    def __init__(self, batch, tokens, kv_heads, head_dim, *, page_size=64, sinks=0, track=False, device="cuda"):
        n = -(-tokens // page_size)
        self.tokens, self.sinks, self.used = tokens, sinks, 0
        self.pages = kv_cache.new_pages((1 + track) * batch * n, kv_heads, head_dim, page_size, device)
        ids = torch.arange((1 + track) * batch * n, dtype=torch.int32, device=device).view(1 + track, batch, n)
        self.table, self.other = ids[0], ids[-1]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.weights = torch.zeros((batch, kv_heads, n * page_size), device=device) if track else None

    def reserve(self, most):
        """Counts at most `most` new tokens of a sequence on the host."""
        if self.used + most > self.tokens:
            raise ValueError(f"the cache holds {self.tokens} tokens, {self.used} + {most} asked for")
        self.used += most

    def grow(self, most, by):
        """Counts new tokens: `by` for each sequence, at most `most`."""
        self.reserve(most)
        try:
            self.lengths += by
        except RuntimeError:
            self.used -= most
            raise

    def append(self, k, v, most, by, offsets=None):
        """Writes new tokens and counts them; where the write is refused, nothing
        is counted."""
        self.grow(most, by)
        try:
            kv_cache.append(self.pages, k, v, self.table, self.lengths, offsets=offsets)
        except Exception:
            self.grow(-most, -by)
            raise

    def evict(self, keep, *, recent=0):
        """Cuts every sequence to its `keep` most attended tokens: the sinks and
        the `recent` last always stay.  Returns the positions they had
        (int32 [batch, kv_heads, keep], -1 past the last)."""
        if self.weights is None:
            raise ValueError("evict needs a cache made with track=True")
        index, kept, lengths = kv_cache.evict(self.pages, self.table, self.lengths, self.weights, keep, self.other,
                                              sinks=self.sinks, recent=recent)
        self.lengths.copy_(lengths)
        old = self.table.clone()
        self.table.copy_(self.other)
        self.other.copy_(old)
        n = min(keep, self.weights.shape[2])
        self.weights[:, :, :n] = kept[:, :, :n]
        self.weights[:, :, n:] = 0
        self.used = min(self.used, keep)
        return index


class MXFP4SelfAttention(nn.Module):
    """q, k, v = x Wqkv^T; y = attention(q, k, v) Wout^T, causal, with an
    optional window and sinks, key heads shared by groups of query heads.

    Both linears are MXFP4Linear (quantized_backward as there).  head_dim =
    dim // heads; 64 or 128 to serve.  Inputs are bf16 or fp16.  q and k
    are taken as they are projected: positions enter with x, or not at all."""

    def __init__(self, dim, heads, kv_heads=None, *, window=None, sinks=0, quantized_backward=False):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        assert dim % heads == 0 and heads % kv_heads == 0, \
            f"dim={dim} must be a multiple of heads={heads}, and heads one of kv_heads={kv_heads}"
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads
        check_mask(window, sinks, None, self.head_dim)
        self.window, self.sinks = window, sinks
        self.qkv = MXFP4Linear(dim, (heads + 2 * kv_heads) * self.head_dim, quantized_backward=quantized_backward)
        self.out = MXFP4Linear(dim, dim, quantized_backward=quantized_backward)
        self.packed = None

    def _split(self, qkv):
        h, g, d = self.heads, self.kv_heads, self.head_dim
        return qkv.unflatten(-1, (h + 2 * g, d)).split((h, g, g), dim=-2)

    def forward(self, x, offsets=None):
        """x [B, T, dim], or with offsets (int32 [B+1]) packed [N, dim]."""
        o = sink_window_attention(*self._split(self.qkv(x)), window=self.window, sinks=self.sinks, offsets=offsets)
        return self.out(o.flatten(-2))

    # -------------------------------------------------------------- serving
    @torch.no_grad()
    def pack(self):
        """Quantizes the weights for prefill and step (again after they change)."""
        self.packed = tuple(quantize_pack_mxfp4(w.weight) for w in (self.qkv, self.out))
        return self

    def new_cache(self, batch, tokens, *, page_size=64, track=False):
        return LayerCache(batch, tokens, self.kv_heads, self.head_dim, page_size=page_size, sinks=self.sinks, track=track,
                          device=self.qkv.weight.device)

    def _served(self):
        if self.packed is None:
            raise RuntimeError("pack() the layer before serving it")
        return self.packed

    @torch.no_grad()
    def prefill(self, x, cache, offsets, longest=None):
        """Prompts packed as [N, dim] into an empty cache; attention is over
        their keys and values before quantization.  longest: the host's bound
        on their lengths (default N).  A cache with track=True takes a second
        pass, over the keys as it holds them, for the prompts' weights."""
        (w, s), (wo, so) = self._served()
        if cache.used:
            raise ValueError("prefill needs an empty cache; step continues one")
        q, k, v = self._split(mxfp4_linear_w(x, w, s))
        cache.append(k, v, x.shape[0] if longest is None else longest, offsets.diff(), offsets)
        o = sink_window_attention(q, k, v, window=self.window, sinks=self.sinks, offsets=offsets)
        if cache.weights is not None and x.shape[0]:
            self._prompt_weights(q, cache, offsets, x.shape[0] if longest is None else longest)
        return mxfp4_linear_w(o.flatten(-2), wo, so)

    def _prompt_weights(self, q, cache, offsets, longest):
        """Adds the weights of packed prompts that fill the cache, the last T tokens
        of every prompt at a time.  Rows before a prompt's first token see nothing."""
        T = max(min(longest, max(64, _WEIGHT_ROWS // max(cache.lengths.numel(), 1))), 1)
        ends = offsets[1:, None].clamp(0, q.shape[0])
        last = ends - T + torch.arange(T, device=q.device)   # token of each row
        for past in range(0, longest, T):
            kv_cache.attend(q[(last - past).clamp(min=0)], cache.pages, cache.table, (cache.lengths - past).clamp(min=0),
                            window=self.window, sinks=self.sinks, weights=cache.weights)

    @torch.no_grad()
    def step(self, x, cache):
        """The next T tokens of every sequence, x [B, T, dim], over the cache."""
        (w, s), (wo, so) = self._served()
        q, k, v = self._split(mxfp4_linear_w(x, w, s))
        cache.append(k, v, x.shape[1], x.shape[1])
        o = kv_cache.attend(q, cache.pages, cache.table, cache.lengths, window=self.window, sinks=self.sinks,
                            weights=cache.weights)
        return mxfp4_linear_w(o.flatten(-2), wo, so)

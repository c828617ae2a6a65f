"""Causal attention with a sliding window and sinks, forward and backward.

The operator between the linears of a transformer block: the reference's
train.py:46-52 calls F.scaled_dot_product_attention there.  Here the rows may
be limited to a window of the last keys, with the first few tokens (sinks)
kept visible, and key heads may be shared by groups of query heads.  Kernels:
lockstep_amd/csrc/attention.hip (forward) and attention_bwd.hip.

Query i of n queries over m keys has position p = i + m - n and sees key j
when 0 <= j <= p and (window is None, or j > p - window, or j < sinks).  A row
that sees nothing gives 0 and takes and passes on no gradient.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _capi as C


def check_mask(window, sinks, scale, head_dim):
    """(window or 0, sinks, scale) as the kernels take them."""
    if window is not None and window < 1:
        raise ValueError(f"window must be None or at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return window or 0, sinks, scale


def rows16(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride along the last axis and 16-byte aligned vectors, else
    a contiguous copy (axes of one element, or none, may have any stride)."""
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16
                      or any(s % 8 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _strides(t: torch.Tensor):
    """(sequence, token, head) strides of a [B, T, H, D] or [N, H, D] tensor."""
    s = [x if n > 1 else 0 for x, n in zip(t.stride(), t.shape)][:-1]
    return (ctypes.c_int64 * 3)(*([0] * (3 - len(s)) + s))


def _args(q, k, v, o, rest, lse, offsets, window, sinks, scale):
    packed = offsets is not None
    return C.Attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), rest.data_ptr() if rest is not None else None,
                       lse.data_ptr(), C.dtype_code(q.dtype), offsets.numel() - 1 if packed else q.shape[0], q.shape[-3], k.shape[-3], q.shape[-2],
                       k.shape[-2], q.shape[-1], _strides(q), _strides(k), _strides(v), _strides(o),
                       offsets.data_ptr() if packed else None, window, sinks, scale)


def _in_reach(t: torch.Tensor, group: int) -> torch.Tensor:
    """rows16(t), its tokens and the heads of a group within the kernels' 32-bit
    offsets."""
    t = rows16(t)
    far = (t.shape[-3] > 1 and t.stride(-3) >= 2 ** 22) or (t.shape[-2] > 1 and t.stride(-2) * group >= 2 ** 29)
    return t.contiguous() if far else t


def _forward(q, k, v, offsets, window, sinks, scale, grad):
    group = q.shape[-2] // k.shape[-2]
    q, k, v = _in_reach(q, group), _in_reach(k, 1), _in_reach(v, 1)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lead = q.shape[:1] if offsets is None else ()
    lse = torch.empty((*lead, q.shape[-2], q.shape[-3]), dtype=torch.float32, device=q.device)
    rest = torch.empty_like(o) if grad else None
    if q.numel():
        a = _args(q, k, v, o, rest, lse, offsets, window, sinks, scale)
        C.call("lsmx_attention_fwd", ctypes.addressof(a), C.stream_of(q))
    return q, k, v, o, rest, lse


class _SinkWindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, window, sinks, scale):
        q, k, v, o, rest, lse = _forward(q, k, v, offsets, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, *(() if offsets is None else (offsets,)))
        ctx.mask = window, sinks, scale
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, _):
        q, k, v, o, rest, lse, *offsets = ctx.saved_tensors
        d_o = _in_reach(d_o.to(q.dtype), q.shape[-2] // k.shape[-2])
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if q.numel() or k.numel():
            a = _args(q, k, v, o, rest, lse, offsets[0] if offsets else None, *ctx.mask)
            n = C.load().lsmx_attention_workspace(ctypes.addressof(a))
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
            st = _strides(d_o)
            C.call("lsmx_attention_bwd", ctypes.addressof(a), d_o.data_ptr(), ctypes.addressof(st), dq.data_ptr(),
                   dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n, C.stream_of(q))
        return dq, dk, dv, None, None, None, None


def sink_window_attention(q, k, v, *, window=None, sinks=0, scale=None, offsets=None, return_lse=False):
    """softmax(scale q k^T) v over the keys each query sees.

    q [B, Tq, H, D], k and v [B, Tk, Hkv, D] (bf16 or fp16; H a multiple of
    Hkv; D a multiple of 8 up to 128; any strides), or with `offsets` (int32
    [B+1], ascending, on the same device) sequences packed along the token
    axis: q [N, H, D], k and v [N, Hkv, D], sequence b being tokens
    offsets[b] .. offsets[b+1]-1; tokens of no sequence see nothing.
    window: keys a query sees, its own the last of them (None: all);
    sinks: first tokens that stay visible past the window; scale: 1/sqrt(D).

    Differentiable in q, k and v (once, in reverse mode).  Scores, softmax and every sum are held in
    fp32; probabilities (and, backward, dS; for dq in two terms) are rounded to
    the inputs' type for the matrix products.  A NaN or infinity in a key that
    a row does not see does not reach the row's result; one in a value may, as
    in a product with weights of 0.  Deterministic.  With return_lse also the natural
    log of each row's softmax sum, fp32 [B, H, Tq] or [H, N] (-inf for a row
    that sees nothing; not differentiable)."""
    if not return_lse and (r := C.fast.attention(q, k, v, offsets, window, sinks, scale)) is not None:
        return r
    C.not_traced("sink_window_attention")
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must share bfloat16 or float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    C.require_device(q, k, v)
    want = 4 if offsets is None else 3
    assert q.dim() == k.dim() == v.dim() == want, f"q, k and v must have {want} axes"
    H, Hkv, D = q.shape[-2], k.shape[-2], q.shape[-1]
    assert k.shape == v.shape and k.shape[-1] == D and (k.shape[0] == q.shape[0]), \
        f"shapes do not match: q {list(q.shape)}, k {list(k.shape)}, v {list(v.shape)}"
    assert H > 0 and Hkv > 0 and H % Hkv == 0, f"H={H} must be a multiple of Hkv={Hkv}"
    assert D % 8 == 0 and 8 <= D <= 128, f"D={D} must be a multiple of 8, 8 to 128"
    if offsets is not None:
        C.require_device(offsets)
        assert offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.numel() >= 1, \
            "offsets must be int32 [B + 1]"
        offsets = offsets.contiguous()
    assert len({t.device for t in (q, k, v, *(() if offsets is None else (offsets,)))}) == 1, \
        "all tensors must be on one device"
    window, sinks, scale = check_mask(window, sinks, scale, D)
    # a dual tensor too goes to the node, which refuses it
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or \
            any(forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v)):
        o, lse = _SinkWindowAttention.apply(q, k, v, offsets, window, sinks, scale)
    else:
        *_, o, _, lse = _forward(q, k, v, offsets, window, sinks, scale, False)
    return (o, lse * math.log(2.0)) if return_lse else o

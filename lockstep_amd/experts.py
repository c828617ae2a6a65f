"""A router and the products of MXFP4 experts.

A mixture of experts keeps most of a model's weights in its experts, and reads
few of them for a token: the place where 4-bit weights save most.  Here the
rows come in MXFP8 (norm.add_rms_norm makes it), the weights in MXFP4
(fp4.quantize_pack_mxfp4 of [E, N, K]), and the matrix instructions take both
as they are:

    y, h, x8, xs = add_rms_norm(x, norm_weight, residual, mxfp8=True)
    weights, ids = route(y @ router.T, k, scoring="sigmoid", bias=b, groups=8, top_groups=4)
    d = dispatch(ids, E)                                  # pairs in the order of their experts
    a8, a_scale = expert_gated(x8, xs, w13, w13_scale, d)  # silu(gate) * up, in MXFP8
    out = expert_combine(a8, a_scale, w2, w2_scale, d, weights)

route is differentiable in the logits; the products, like the weight-only ones
(mxfp4_gemm.mxfp4_linear_w), are not.  No call synchronizes.  Kernels:
lockstep_amd/csrc/route.hip and experts.hip.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _capi as C


class Dispatch(NamedTuple):
    """experts int32 [.., k]: each token's experts (any other number: none);
    order int32 [tokens * k]: the pairs token * k + slot sorted by expert,
    stable, those of no expert last; offsets int32 [E + 1]: expert e's pairs
    are order[offsets[e]] .. order[offsets[e + 1] - 1]."""
    experts: torch.Tensor
    order: torch.Tensor
    offsets: torch.Tensor


# ------------------------------------------------------------------- router
def _route_args(logits, opts, weights, ids, bias, mask):
    k, sigmoid, groups, top_groups, renorm, scale = opts
    return C.Route(logits.data_ptr(), C.dtype_code(logits.dtype), logits.shape[0],
                   logits.stride(0) if logits.shape[0] > 1 else logits.shape[1], logits.shape[1], k, sigmoid, groups,
                   top_groups, renorm, scale, None if bias is None else bias.data_ptr(),
                   None if mask is None else mask.data_ptr(), None if weights is None else weights.data_ptr(), ids.data_ptr())


def _route(logits, bias, mask, opts):
    rows, k = logits.shape[0], opts[0]
    weights = torch.empty((rows, k), dtype=torch.float32, device=logits.device)
    ids = torch.empty((rows, k), dtype=torch.int32, device=logits.device)
    if rows:
        a = _route_args(logits, opts, weights, ids, bias, mask)
        with C.on_device_of(logits):
            C.call("lsmx_route_fwd", ctypes.addressof(a), C.stream_of(logits))
    return weights, ids


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, mask, opts):
        weights, ids = _route(logits, bias, mask, opts)
        ctx.save_for_backward(logits, ids)
        ctx.opts = opts
        ctx.mark_non_differentiable(ids)
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dw, _):
        logits, ids = ctx.saved_tensors
        dl = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if dl.numel():
            dw = dw.float().contiguous()
            a = _route_args(logits, ctx.opts, None, ids, None, None)
            with C.on_device_of(logits):
                C.call("lsmx_route_bwd", ctypes.addressof(a), dw.data_ptr(), dl.data_ptr(), C.stream_of(logits))
        return dl, None, None, None


def route(logits, k, *, bias=None, scoring="softmax", groups=1, top_groups=1, renormalize=True, scale=1.0, mask=None):
    """The k experts of every token, and their weights.

    logits [.., E] (fp32, bf16 or fp16; E up to 1024).  The scores s are
    softmax(logits) or, scoring="sigmoid", 1 / (1 + exp(-logits)).  Experts are
    ranked by s + bias (fp32 [E]; balances their load, does not enter the
    weights).  With groups > 1 (equal runs of experts, up to 64) only the
    top_groups whose two largest ranks have the largest sums take part.
    Returns (weights fp32 [.., k], experts int32 [.., k]), the largest rank first,
    ties (of groups too) to the lowest index; ranks are compared in 64 bits,
    without a bias as their logits, which have the scores' order.
    The weights are s of the chosen, with renormalize=True divided by their
    sum (0 where that is 0), times scale.

    mask (bool [..]): tokens with False, such as padding, get experts -1 and
    weights 0.  A NaN ranks first; a row of nothing but -inf scores 0.
    Differentiable in logits (once, in reverse mode): the choice is taken as
    given, and neither it nor bias has a gradient.  A differentiable call is not
    captured into a HIP graph while an eager graph of the logits, made on the
    default stream, is alive."""
    if (r := C.fast.route(logits, k, bias, scoring, groups, top_groups, renormalize, scale, mask)) is not None:
        return r
    C.not_traced("route")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    given = [t for t in (logits, bias, mask) if t is not None]
    C.require_device(*given)
    C.one_device(*given)
    assert logits.dim() >= 1, "logits must be [.., E]"
    E, lead = logits.shape[-1], logits.shape[:-1]
    assert 1 <= E <= 1024, f"E={E} must be 1 to 1024"
    if not (1 <= groups <= 64 and E % groups == 0 and 1 <= top_groups <= groups):
        raise ValueError(f"groups={groups} must be 1 to 64 and divide E={E}, top_groups={top_groups} be 1 to groups")
    if not 1 <= k <= min(64, E // groups * top_groups):
        raise ValueError(f"k={k} must be 1 to 64 and at most the {E // groups * top_groups} experts that take part")
    scale = float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if bias is not None:
        assert bias.dtype == torch.float32 and bias.shape == (E,), f"bias must be float32 [{E}]"
        bias = bias.detach().contiguous()
    if mask is not None:
        assert mask.dtype == torch.bool and mask.shape == lead, f"mask must be bool {list(lead)}"
        mask = mask.contiguous()
    l2 = logits.reshape(-1, E) if E else logits
    if (l2.stride(1) != 1 and E > 1) or (l2.shape[0] > 1 and l2.stride(0) < E):
        l2 = l2.contiguous()
    opts = (int(k), int(scoring == "sigmoid"), int(groups), int(top_groups), int(bool(renormalize)), scale)
    # a dual tensor too goes to the node, which refuses it
    if (torch.is_grad_enabled() and logits.requires_grad) or forward_ad.unpack_dual(logits).tangent is not None:
        C.fast.captures((l2,), None)
        weights, ids = _Route.apply(l2, bias, mask, opts)
    else:
        weights, ids = _route(l2, bias, mask, opts)
    return weights.view(*lead, k), ids.view(*lead, k)


# ----------------------------------------------------------------- products
def dispatch(experts, num_experts) -> Dispatch:
    """The (token, slot) pairs of experts (int32 [.., k]) in the order of their
    experts, for expert_gated and expert_combine.  Ids outside
    0 .. num_experts - 1 (up to 1024 experts) stand for no expert.  Up to 2^21
    pairs."""
    if (r := C.fast.dispatch(experts, num_experts)) is not None:
        return Dispatch(experts, *r)
    C.not_traced("dispatch")
    C.require_device(experts)
    assert experts.dtype == torch.int32 and experts.dim() >= 1, f"experts must be int32 [.., k], got {experts.dtype}"
    assert 1 <= num_experts <= 1024, f"num_experts={num_experts} must be 1 to 1024"
    assert experts.numel() <= 2 ** 21, f"{experts.numel()} pairs, at most 2^21"
    ids = experts.contiguous()
    order = torch.empty(ids.numel(), dtype=torch.int32, device=ids.device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=ids.device)
    n = C.load().lsmx_dispatch_workspace(ids.numel(), num_experts)
    ws = torch.empty(n, dtype=torch.uint8, device=ids.device) if n else None
    with C.on_device_of(ids):
        C.call("lsmx_dispatch", ids.data_ptr(), ids.numel(), num_experts, order.data_ptr(), offsets.data_ptr(),
               None if ws is None else ws.data_ptr(), n, C.stream_of(ids))
    return Dispatch(ids, order, offsets)


def _dense16(t):
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _check(x, x_scale, w, w_scale, d, lead, more=()):
    """The C description of a product over rows x [*lead, K], its tensors checked."""
    C.require_device(x, x_scale, w, w_scale, *d, *more)
    C.one_device(x, x_scale, w, w_scale, *d, *more)
    if x.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError(f"rows must be float8_e4m3fn codes, got {x.dtype}")
    if x_scale.dtype != torch.uint8 or w.dtype != torch.uint8 or w_scale.dtype != torch.uint8:
        raise TypeError("scales must be E8M0 bytes (uint8), weights packed MXFP4 (uint8)")
    assert w.dim() == 3 and w.shape[0] >= 1, "weights must be [E, N, K // 2]"
    E, N, half = w.shape
    K = 2 * half
    assert K % 128 == 0 and K > 0, f"K={K} must be a multiple of 128"
    assert w_scale.shape == (E, N, K // 32), f"w_scale must be {[E, N, K // 32]}, got {list(w_scale.shape)}"
    assert d.experts.dtype == d.order.dtype == d.offsets.dtype == torch.int32 and d.experts.dim() >= 1 and \
        d.order.shape == (d.experts.numel(),) and d.offsets.shape == (E + 1,), \
        f"d must be dispatch(experts, {E}): order [{d.experts.numel()}], offsets [{E + 1}]"
    assert x.shape == (*lead, K), f"rows must be {[*lead, K]}, got {list(x.shape)}"
    assert x_scale.shape == (*lead, K // 32), f"their scales must be {[*lead, K // 32]}, got {list(x_scale.shape)}"
    k = d.experts.shape[-1]
    assert 1 <= k <= 1024 and E <= 1024 and d.experts.numel() <= 2 ** 21, "up to 1024 experts, 1024 slots, 2^21 pairs"
    assert N * K // 2 < 2 ** 31 and N > 0, "an expert's weights must stay below 2^31 bytes"
    keep = [_dense16(t) for t in (x, x_scale, w, w_scale, *d)]
    a = C.Experts(*(t.data_ptr() for t in keep), d.experts.numel() // k, k, E, N, K)
    return a, keep, N


def expert_gated(x, x_scale, w, w_scale, d):
    """silu(x Wg^T) * (x Wu^T) of every token's row with each of its experts.

    x [.., K] float8_e4m3fn codes with x_scale [.., K // 32] E8M0 bytes: MXFP8,
    as add_rms_norm(mxfp8=True) gives it.  w [E, 2 F, K // 2] packed MXFP4
    with w_scale [E, 2 F, K // 32], rows 0 .. F - 1 the gate's (Wg), the others
    up's; K a multiple of 128, F of 32.  d: dispatch(experts [.., k], E).
    Returns (h float8_e4m3fn [.., k, F], h_scale uint8 [.., k, F // 32]) in
    MXFP8; zeros for slots of no expert.  The matrix instruction adds eight
    products at a time and keeps 13 bits below the largest exponent among them
    (an error below 7 * 2^-13 of the summed magnitudes, 4e-6 of a result on
    normal values), the eights are added in fp32; up to 4 rows for an expert
    on average nothing is lost within the eight.  The gate is fp32, h is rounded
    once.  No gradient."""
    if (r := C.fast.expert_gated(x, x_scale, w, w_scale, d)) is not None:
        return r
    C.not_traced("expert_gated")
    a, keep, N = _check(x, x_scale, w, w_scale, d, d.experts.shape[:-1])
    assert N % 64 == 0, f"w must hold 2 F rows, F a multiple of 32, got {N}"
    h = torch.empty((*d.experts.shape, N // 2), dtype=torch.float8_e4m3fn, device=x.device)
    hs = torch.empty((*d.experts.shape, N // 64), dtype=torch.uint8, device=x.device)
    if h.numel():
        with C.on_device_of(x):
            C.call("lsmx_expert_gated", ctypes.addressof(a), h.data_ptr(), hs.data_ptr(), C.stream_of(x))
    return h, hs


def expert_combine(h, h_scale, w, w_scale, d, weights, out_dtype=torch.bfloat16):
    """y = sum over a token's slots of weights times h W^T with the slot's expert.

    h [.., k, K] and h_scale [.., k, K // 32]: MXFP8, as expert_gated gives them.
    w [E, N, K // 2] packed MXFP4 with w_scale [E, N, K // 32]; K a multiple of
    128.  weights fp32 [.., k], as route gives them.  Returns y [.., N] in
    out_dtype (bf16, fp16 or fp32).  Slots of no expert add nothing.
    Products are as expert_gated's, sums are fp32, a token's slots are added in
    their order, y is rounded once: results do not depend on the run.  For y in
    bf16 with many rows for an expert (more than 24 on average) each slot's row
    is rounded to 11 bits before the sum, an eighth of y's own rounding.  No
    gradient."""
    if (r := C.fast.expert_combine(h, h_scale, w, w_scale, d, weights, out_dtype)) is not None:
        return r
    C.not_traced("expert_combine")
    code = C.dtype_code(out_dtype)
    a, keep, N = _check(h, h_scale, w, w_scale, d, d.experts.shape, (weights,))
    assert weights.dtype == torch.float32 and weights.shape == d.experts.shape, \
        f"weights must be float32 {list(d.experts.shape)}"
    weights = weights.detach().contiguous()
    y = torch.empty((*d.experts.shape[:-1], N), dtype=out_dtype, device=h.device)
    if y.numel():
        n = C.load().lsmx_expert_combine_workspace(ctypes.addressof(a))
        ws = torch.empty(n, dtype=torch.uint8, device=h.device)
        with C.on_device_of(h):
            C.call("lsmx_expert_combine", ctypes.addressof(a), weights.data_ptr(), y.data_ptr(), code, ws.data_ptr(), n,
                   C.stream_of(h))
    return y

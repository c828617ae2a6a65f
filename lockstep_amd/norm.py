"""Root-mean-square norm with the residual's addition, forward and backward.

What stands before the linears of a block: the residual stream takes the last
layer's output, and its norm goes on in x's type and, for the block-scaled
products (mxfp4_gemm.mxfp4_gemm_fp8 with E8M0 scales, experts.expert_gated), in
MXFP8 as well.  Kernels: lockstep_amd/csrc/norm.hip.

MXFP8 here: E4M3 codes with one E8M0 scale for 32 elements along the row, the
least power of two that keeps the block within 448 (no element saturates), 1
for a block of zeros, NaN for a block with an infinity or a NaN.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _capi as C


def _rows(t: torch.Tensor, aligned: bool) -> torch.Tensor:
    """t [.., D] as rows of unit stride that do not overlap, else a contiguous
    copy; with `aligned`, rows of 16-byte aligned vectors."""
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]) or (
            aligned and (t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) * t.element_size() % 16))):
        t = t.contiguous()
        if aligned and t.data_ptr() % 16:
            t = t.clone()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, w, r, eps, mxfp8):
    """(x's rows, y, h, codes, scale), y and h in x's shape."""
    x2, r2 = _rows(x, mxfp8), None if r is None else _rows(r, mxfp8)
    w = w.clone() if mxfp8 and w.data_ptr() % 16 else w
    D = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = None if r is None else torch.empty_like(y)
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device) if mxfp8 else None
    scale = torch.empty((*x.shape[:-1], D // 32), dtype=torch.uint8, device=x.device) if mxfp8 else None
    if x.numel():
        with C.on_device_of(x):
            C.call("lsmx_rms_norm", x2.data_ptr(), _ld(x2), _ptr(r2), 0 if r is None else _ld(r2), C.dtype_code(x.dtype),
                   w.data_ptr(), C.dtype_code(w.dtype), x2.shape[0], D, eps, _ptr(h), y.data_ptr(), _ptr(codes),
                   _ptr(scale), C.stream_of(x))
    return x2, y, h, codes, scale


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, r, eps, mxfp8):
        x2, y, h, codes, scale = _forward(x, w, r, eps, mxfp8)
        ctx.save_for_backward(x2 if r is None else h, w)
        ctx.eps, ctx.residual = eps, r is not None
        ctx.set_materialize_grads(False)
        if mxfp8:
            ctx.mark_non_differentiable(codes, scale)
        return y, h, codes, scale

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh, *_):
        h, w = ctx.saved_tensors
        if dy is None:
            return dh, None, dh if ctx.residual else None, None, None
        D = h.shape[-1]
        dx = torch.empty(dy.shape, dtype=h.dtype, device=h.device)
        dw = torch.empty_like(w) if ctx.needs_input_grad[1] else None
        if dx.numel() == 0:
            return dx, None if dw is None else dw.zero_(), dx if ctx.residual else None, None, None
        h2, dy2 = _rows(h, False), _rows(dy.to(h.dtype), False)
        dh2 = None if dh is None else _rows(dh.to(h.dtype), False)
        n = C.load().lsmx_rms_norm_bwd_workspace(h2.shape[0], D, C.dtype_code(h.dtype)) if dw is not None else 0
        ws = torch.empty(n, dtype=torch.uint8, device=h.device) if n else None
        with C.on_device_of(h):
            C.call("lsmx_rms_norm_bwd", h2.data_ptr(), _ld(h2), dy2.data_ptr(), _ld(dy2), _ptr(dh2),
                   0 if dh is None else _ld(dh2), C.dtype_code(h.dtype), w.data_ptr(), C.dtype_code(w.dtype), h2.shape[0], D,
                   ctx.eps, dx.data_ptr(), _ptr(dw), _ptr(ws), n, C.stream_of(h))
        return dx, dw, dx if ctx.residual else None, None, None


def add_rms_norm(x, weight, residual=None, *, eps=1e-6, mxfp8=False):
    """h = x + residual, rounded to their type, and y = h / sqrt(mean(h^2) + eps) * weight.

    x and residual [.., D] (fp32, bf16 or fp16, one type and shape, any
    strides), weight [D] of that type or fp32.  Returns y, or with a residual
    (y, h); with mxfp8=True (D a multiple of 32) two more: y as it was before
    rounding in MXFP8, codes (float8_e4m3fn [.., D]) and E8M0 scales (uint8
    [.., D // 32]), the row-major form that mxfp4_gemm_fp8 takes.

    Differentiable in x, residual and weight (once, in reverse mode; the
    codes have no gradient).  The mean, the norm and every sum are fp32; y is
    rounded once, its codes are of the unrounded y.  Deterministic.  A
    differentiable call is not captured into a HIP graph while an eager graph of
    its tensors, made on the default stream, is alive."""
    if (r := C.fast.rms_norm(x, weight, residual, eps, mxfp8)) is not None:
        return r
    C.not_traced("add_rms_norm")
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if residual is not None and residual.dtype != x.dtype:
        raise TypeError(f"x and residual must share a type, got {x.dtype}, {residual.dtype}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    both = (x, weight) if residual is None else (x, weight, residual)
    C.require_device(*both)
    C.one_device(*both)
    assert x.dim() >= 1 and x.shape[-1] > 0, "x must be [.., D], D at least 1"
    assert weight.shape == x.shape[-1:], f"weight must be [{x.shape[-1]}], got {list(weight.shape)}"
    assert residual is None or residual.shape == x.shape, \
        f"x and residual must have one shape, got {list(x.shape)}, {list(residual.shape)}"
    assert not mxfp8 or x.shape[-1] % 32 == 0, f"D={x.shape[-1]} must be a multiple of 32 for MXFP8"
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    weight = weight.contiguous()
    # a dual tensor too goes to the node, which refuses it
    if (torch.is_grad_enabled() and any(t.requires_grad for t in both)) or \
            any(forward_ad.unpack_dual(t).tangent is not None for t in both):
        C.fast.captures(both, None)
        y, h, codes, scale = _AddRMSNorm.apply(x, weight, residual, eps, bool(mxfp8))
    else:
        _, y, h, codes, scale = _forward(x, weight, residual, eps, bool(mxfp8))
    got = tuple(t for t in (y, h, codes, scale) if t is not None)
    return got if len(got) > 1 else y

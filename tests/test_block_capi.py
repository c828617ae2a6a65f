"""What the norm, the router and the experts' products refuse: through the C
ABI before any device is touched, and through the Python functions."""

import ctypes

import pytest
import torch

from lockstep_amd import _capi as C
from lockstep_amd import experts, norm

P = 0x1000   # never dereferenced: validation fails first


def rc(name, *args):
    return getattr(C.load(), name)(*args)


def rms(**k):
    a = dict(x=P, ldx=64, r=P, ldr=64, dtype=C.BF16, w=P, w_dtype=C.BF16, rows=4, dim=64, eps=1e-6, h=P, y=P, codes=P, scale=P)
    a.update(k)
    return rc("lsmx_rms_norm", *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=7), C.ERR_DTYPE), (dict(w_dtype=C.F16), C.ERR_DTYPE), (dict(rows=-1), C.ERR_SHAPE), (dict(dim=1 << 31), C.ERR_SHAPE),
    (dict(eps=-1.0), C.ERR_ARG), (dict(eps=float("nan")), C.ERR_ARG), (dict(eps=float("inf")), C.ERR_ARG), (dict(x=None), C.ERR_ARG),
    (dict(w=None), C.ERR_ARG), (dict(y=None), C.ERR_ARG), (dict(h=None), C.ERR_ARG), (dict(codes=None), C.ERR_ARG),
    (dict(scale=None), C.ERR_ARG), (dict(ldx=63), C.ERR_SHAPE), (dict(ldr=63), C.ERR_SHAPE), (dict(x=P + 1), C.ERR_ALIGN),
    (dict(w=P + 2, w_dtype=C.F32), C.ERR_ALIGN), (dict(x=P + 2), C.ERR_ALIGN), (dict(ldx=65), C.ERR_ALIGN), (dict(codes=P + 4), C.ERR_ALIGN),
    (dict(dim=48), C.ERR_SHAPE)])
def test_norm_refusals(change, code):
    assert rms(**change) == code
    assert "lsmx_rms_norm" in C.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), C.ERR_DTYPE), (dict(rows=0), C.ERR_SHAPE), (dict(h=None), C.ERR_ARG), (dict(dy=None), C.ERR_ARG),
    (dict(dx=None), C.ERR_ARG), (dict(ws=None), C.ERR_ARG), (dict(ws_bytes=4 * 64 * 4 - 1), C.ERR_ARG), (dict(ldh=1), C.ERR_SHAPE),
    (dict(lddy=1), C.ERR_SHAPE), (dict(lddh=1), C.ERR_SHAPE), (dict(dw=P + 1), C.ERR_ALIGN), (dict(ws=P + 8), C.ERR_ALIGN)])
def test_norm_backward_refusals(change, code):
    a = dict(h=P, ldh=64, dy=P, lddy=64, dh=P, lddh=64, dtype=C.BF16, w=P, w_dtype=C.BF16, rows=4, dim=64, eps=1e-6, dx=P, dw=P, ws=P,
             ws_bytes=4 * 64 * 4)
    assert rc("lsmx_rms_norm_bwd_workspace", 4, 64, C.BF16) <= a["ws_bytes"]
    a.update(change)
    if "ws_bytes" in change:
        a["ws_bytes"] = rc("lsmx_rms_norm_bwd_workspace", 4, 64, C.BF16) - 1
    assert rc("lsmx_rms_norm_bwd", *a.values(), None) == code


def route(**k):
    a = dict(logits=P, dtype=C.F32, rows=4, ld=64, experts=64, k=4, sigmoid=0, groups=8, top_groups=2, renorm=1, scale=1.0, bias=P,
             mask=P, weights=P, ids=P)
    a.update(k)
    return C.Route(*a.values())


ROUTE = [(dict(dtype=5), C.ERR_DTYPE), (dict(experts=0), C.ERR_SHAPE), (dict(experts=1025, ld=1025, groups=1, top_groups=1), C.ERR_SHAPE),
         (dict(groups=0), C.ERR_SHAPE), (dict(groups=7), C.ERR_SHAPE), (dict(groups=128, experts=128, ld=128), C.ERR_SHAPE),
         (dict(top_groups=0), C.ERR_SHAPE), (dict(top_groups=9), C.ERR_SHAPE), (dict(k=0), C.ERR_SHAPE), (dict(k=17), C.ERR_SHAPE),
         (dict(experts=1024, ld=1024, k=65), C.ERR_SHAPE), (dict(rows=-1), C.ERR_SHAPE), (dict(ld=63), C.ERR_SHAPE),
         (dict(scale=0.0), C.ERR_ARG), (dict(scale=float("nan")), C.ERR_ARG), (dict(logits=None), C.ERR_ARG), (dict(ids=None), C.ERR_ARG),
         (dict(bias=P + 2), C.ERR_ALIGN), (dict(logits=P + 2), C.ERR_ALIGN)]


@pytest.mark.parametrize("change,code", ROUTE + [(dict(weights=None), C.ERR_ARG)])
def test_route_refusals(change, code):
    a = route(**change)
    assert rc("lsmx_route_fwd", ctypes.addressof(a), None) == code


@pytest.mark.parametrize("change,code", ROUTE)
def test_route_backward_refusals(change, code):
    a = route(**change)
    assert rc("lsmx_route_bwd", ctypes.addressof(a), P, P, None) == code


def test_route_null_arguments():
    a = route()
    assert rc("lsmx_route_fwd", None, None) == C.ERR_ARG and rc("lsmx_route_bwd", None, P, P, None) == C.ERR_ARG
    assert rc("lsmx_route_bwd", ctypes.addressof(a), None, P, None) == C.ERR_ARG
    assert rc("lsmx_route_bwd", ctypes.addressof(a), P, None, None) == C.ERR_ARG


def test_dispatch_refusals():
    big = 1 << 20
    n = rc("lsmx_dispatch_workspace", big, 64)
    assert n > 0 and rc("lsmx_dispatch_workspace", 8, 64) == 0
    assert rc("lsmx_dispatch", P, 8, 0, P, P, None, 0, None) == C.ERR_SHAPE
    assert rc("lsmx_dispatch", P, 8, 1025, P, P, None, 0, None) == C.ERR_SHAPE
    assert rc("lsmx_dispatch", P, (1 << 21) + 1, 64, P, P, P, 1 << 30, None) == C.ERR_SHAPE
    assert rc("lsmx_dispatch", P, -1, 64, P, P, None, 0, None) == C.ERR_SHAPE
    assert rc("lsmx_dispatch", None, 8, 64, P, P, None, 0, None) == C.ERR_ARG
    assert rc("lsmx_dispatch", P, 8, 64, None, P, None, 0, None) == C.ERR_ARG
    assert rc("lsmx_dispatch", P, 8, 64, P, None, None, 0, None) == C.ERR_ARG
    assert rc("lsmx_dispatch", P, big, 64, P, P, None, n, None) == C.ERR_ARG
    assert rc("lsmx_dispatch", P, big, 64, P, P, P, n - 1, None) == C.ERR_ARG
    assert rc("lsmx_dispatch", P + 2, 8, 64, P, P, None, 0, None) == C.ERR_ALIGN


def product(**k):
    a = dict(x=P, x_scale=P, w=P, w_scale=P, ids=P, order=P, offsets=P, tokens=8, k=2, experts=4, N=128, K=256)
    a.update(k)
    return C.Experts(*a.values())


PRODUCT = [(dict(x=None), C.ERR_ARG), (dict(x_scale=None), C.ERR_ARG), (dict(w=None), C.ERR_ARG), (dict(w_scale=None), C.ERR_ARG),
           (dict(ids=None), C.ERR_ARG), (dict(order=None), C.ERR_ARG), (dict(offsets=None), C.ERR_ARG), (dict(tokens=-1), C.ERR_SHAPE),
           (dict(tokens=1 << 21), C.ERR_SHAPE), (dict(k=0), C.ERR_SHAPE), (dict(k=1025), C.ERR_SHAPE), (dict(experts=0), C.ERR_SHAPE),
           (dict(experts=1025), C.ERR_SHAPE), (dict(K=0), C.ERR_SHAPE), (dict(K=192), C.ERR_SHAPE), (dict(N=0), C.ERR_SHAPE),
           (dict(N=1 << 20, K=4096), C.ERR_SHAPE), (dict(x=P + 8), C.ERR_ALIGN), (dict(w=P + 8), C.ERR_ALIGN),
           (dict(w_scale=P + 1), C.ERR_ALIGN), (dict(order=P + 2), C.ERR_ALIGN)]


@pytest.mark.parametrize("change,code", PRODUCT + [(dict(N=96), C.ERR_SHAPE)])
def test_gated_refusals(change, code):
    a = product(**change)
    assert rc("lsmx_expert_gated", ctypes.addressof(a), P, P, None) == code


@pytest.mark.parametrize("change,code", PRODUCT)
def test_combine_refusals(change, code):
    a = product(**change)
    assert rc("lsmx_expert_combine", ctypes.addressof(a), P, P, C.BF16, P, 1 << 40, None) == code


def test_product_null_arguments():
    a = product()
    at, n = ctypes.addressof(a), rc("lsmx_expert_combine_workspace", ctypes.addressof(a))
    assert rc("lsmx_expert_gated", None, P, P, None) == C.ERR_ARG and rc("lsmx_expert_gated", at, None, P, None) == C.ERR_ARG
    assert rc("lsmx_expert_gated", at, P, None, None) == C.ERR_ARG and rc("lsmx_expert_gated", at, P + 2, P, None) == C.ERR_ALIGN
    assert rc("lsmx_expert_combine", at, None, P, C.BF16, P, n, None) == C.ERR_ARG
    assert rc("lsmx_expert_combine", at, P, None, C.BF16, P, n, None) == C.ERR_ARG
    assert rc("lsmx_expert_combine", at, P, P, C.BF16, None, n, None) == C.ERR_ARG
    assert rc("lsmx_expert_combine", at, P, P, C.BF16, P, n - 1, None) == C.ERR_ARG
    assert rc("lsmx_expert_combine", at, P, P, C.E4M3, P, n, None) == C.ERR_DTYPE


# -------------------------------------------------------- the Python functions
def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64), torch.zeros(64)
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    d = experts.Dispatch(i32(4, 2), i32(8), i32(3))
    for call in (lambda: norm.add_rms_norm(x, w), lambda: experts.route(x, 2), lambda: experts.dispatch(i32(4, 2), 4),
                 lambda: experts.expert_gated(u8(4, 128), u8(4, 4), u8(2, 64, 64), u8(2, 64, 4), d),
                 lambda: experts.expert_combine(u8(4, 2, 128), u8(4, 2, 4), u8(2, 64, 64), u8(2, 64, 4), d, x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_types_are_refused():
    w = torch.zeros(64)
    with pytest.raises(TypeError, match="x must be"):
        norm.add_rms_norm(torch.zeros(4, 64, dtype=torch.float64), w)
    with pytest.raises(TypeError, match="share a type"):
        norm.add_rms_norm(torch.zeros(4, 64), w, torch.zeros(4, 64, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="weight must be"):
        norm.add_rms_norm(torch.zeros(4, 64, dtype=torch.bfloat16), w.half())
    with pytest.raises(TypeError, match="logits must be"):
        experts.route(torch.zeros(4, 64, dtype=torch.float64), 2)
    with pytest.raises(ValueError, match="scoring"):
        experts.route(torch.zeros(4, 64), 2, scoring="top")


@pytest.mark.gpu
def test_arguments_are_refused_on_the_gpu(dev):
    x, w = torch.zeros((4, 64), device=dev), torch.zeros(64, device=dev)
    for bad in (dict(weight=w[:32]), dict(residual=x[:3]), dict(x=x[:, :40], weight=w[:40], mxfp8=True)):
        with pytest.raises(AssertionError):
            norm.add_rms_norm(**{"x": x, "weight": w, **bad})
    with pytest.raises(ValueError, match="eps"):
        norm.add_rms_norm(x, w, eps=-1)
    with pytest.raises(RuntimeError, match="twice|does not require grad"):
        a = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(norm.add_rms_norm(a, w).sum(), a, create_graph=True)
        g.sum().backward()
    for bad in (dict(k=0), dict(k=65), dict(groups=3), dict(groups=4, top_groups=5), dict(k=17, groups=4), dict(scale=0), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            experts.route(x, **{"k": 2, **bad})
    for bad in (dict(bias=w.bfloat16()), dict(bias=w[:3]), dict(mask=torch.ones(4, device=dev)), dict(mask=torch.ones(3, dtype=torch.bool, device=dev))):
        with pytest.raises(AssertionError):
            experts.route(x, 2, **bad)
    ids = torch.zeros((4, 2), dtype=torch.int32, device=dev)
    for bad in ((ids.long(), 4), (ids, 0), (ids, 1025)):
        with pytest.raises(AssertionError):
            experts.dispatch(*bad)
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device=dev)  # noqa: E731
    d = experts.dispatch(ids, 2)
    good = dict(x=u8(4, 128), x_scale=u8(4, 4), w=u8(2, 64, 64), w_scale=u8(2, 64, 4), d=d)
    experts.expert_gated(**good)
    for bad in (dict(x=u8(3, 128)), dict(x=u8(4, 256)), dict(x_scale=u8(4, 3)), dict(w=u8(2, 32, 64), w_scale=u8(2, 32, 4)),
                dict(w=u8(2, 64, 48), w_scale=u8(2, 64, 3), x=u8(4, 96), x_scale=u8(4, 3)), dict(w_scale=u8(2, 64, 3)),
                dict(w=u8(3, 64, 64), w_scale=u8(3, 64, 4)), dict(d=d._replace(order=d.order[:7])), dict(d=d._replace(experts=ids.long()))):
        with pytest.raises(AssertionError):
            experts.expert_gated(**{**good, **bad})
    with pytest.raises(TypeError):
        experts.expert_gated(**{**good, "x": good["x"].float()})
    with pytest.raises(TypeError):
        experts.expert_gated(**{**good, "x_scale": good["x_scale"].float()})
    good = dict(h=u8(4, 2, 128), h_scale=u8(4, 2, 4), w=u8(2, 64, 64), w_scale=u8(2, 64, 4), d=d, weights=torch.zeros((4, 2), device=dev))
    experts.expert_combine(**good)
    for bad in (dict(h=u8(4, 128)), dict(weights=torch.zeros((4, 2), device=dev).half()), dict(weights=torch.zeros(4, device=dev))):
        with pytest.raises(AssertionError):
            experts.expert_combine(**{**good, **bad})
    with pytest.raises(TypeError):
        experts.expert_combine(**good, out_dtype=torch.float64)


@pytest.mark.parametrize("change,ok", [(dict(tokens=1 << 21, k=1, K=256, N=1 << 10), True), (dict(tokens=1 << 21, k=1, K=256, N=1 << 12), False),
                                       (dict(tokens=1 << 21, k=1, K=512, N=1 << 13), True), (dict(tokens=1 << 21, k=1, K=512, N=1 << 16), False),
                                       (dict(tokens=1 << 21, k=1, K=512, N=14336), False), (dict(tokens=1 << 20, k=2, K=512, N=14336), True)])
def test_launches_past_their_limit_are_refused(change, ok):
    """2^32 threads: the workspace's size is 0 for a refused call."""
    a = product(**change)
    n = rc("lsmx_expert_combine_workspace", ctypes.addressof(a))
    assert (n > 0) == ok
    if not ok:
        assert rc("lsmx_expert_combine", ctypes.addressof(a), P, P, C.BF16, P, 1 << 50, None) == C.ERR_SHAPE
        assert "too many" in C.last_error()


def test_gated_needs_aligned_rows():
    a = product()
    assert rc("lsmx_expert_gated", ctypes.addressof(a), P + 4, P, None) == C.ERR_ALIGN


@pytest.mark.parametrize("src", ["norm.hip", "route.hip", "experts.hip"])
def test_kernels_use_no_scratch(src, tmp_path):
    """The products count their loads in flight, which a spill would add to."""
    from .test_kernel_resources import test_kernels_use_no_scratch as check
    check(src, tmp_path)

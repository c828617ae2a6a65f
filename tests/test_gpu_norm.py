"""norm.add_rms_norm against its formula in 64 bits.

Bounds, for u = half a step of the output's type: the mean, its root and the
products are fp32, a sum of n terms in a tree of threads of at most n / 64 + 16
additions each, so a value v carries at most u |v| + 2^-18 of the magnitudes
that are added up for it (n <= 32768 here adds 528 of 2^-24, 2^-15, to the mean,
half of it to its root: sums of squares have no cancellation and round at
random, 2^-18 holds with a margin of 8).  E4M3 rounds by 2^-4 of a normal value,
by half of 2^-9 of the scale below."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -18


def _u(dt):
    return torch.finfo(dt).eps / 2


def _inputs(dev, T, D, dt, seed, w_dt=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    wide = torch.exp(torch.randn(D, generator=g, device=dev))
    x = torch.randn((T, D), generator=g, device=dev).to(dt)
    r = (torch.randn((T, D), generator=g, device=dev) * wide).to(dt)
    w = (1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(w_dt or dt)
    return x, r, w


def _exact(h, w, eps):
    h = h.double()
    inv = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h * inv * w.double(), inv


def _check_mx8(codes, scale, y):
    """codes and scales against the unrounded y in 64 bits."""
    b = y.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.ceil(torch.log2(torch.where(top == 0, 448.0, top) / 448)).clamp(min=-127)
    near = torch.ceil(torch.log2(top * (1 + 1e-5) / 448)) != torch.ceil(torch.log2(top * (1 - 1e-5) / 448))
    got = scale.double() - 127
    assert torch.equal(got[~near], e[~near]) and ((got - e).abs() <= 1).all()
    s = torch.exp2(got)[..., None]
    v = codes.double().unflatten(-1, (-1, 32)) * s
    assert ((v - b).abs() <= b.abs() * (2.0 ** -4 + TINY) + s * 2.0 ** -10 * (1 + TINY) + b.abs().amax(-1, keepdim=True) * 2.0 ** -22).all()


# dims: one element, below and past a vector, odd, the forms' limits and past them
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,D", [(1, 1), (3, 7), (2, 8), (5, 33), (9, 512), (7, 520), (4, 1000), (3, 1024), (5, 2048),
                                 (3, 2049), (2, 4096), (2, 4100), (3, 8192), (2, 8193), (2, 16384), (1, 32768), (2, 32776)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(dev, dt, T, D, residual):
    from lockstep_amd.norm import add_rms_norm
    dt = DT[dt]
    x, r, w = _inputs(dev, T, D, dt, 7 * D + T, torch.float32 if D % 3 == 0 else None)
    if residual:
        y, h = add_rms_norm(x, w, r, eps=1e-5)
        assert torch.equal(h, (x.float() + r.float()).to(dt))
    else:
        h, y = x, add_rms_norm(x, w, eps=1e-5)
    want, _ = _exact(h, w, 1e-5)
    assert y.dtype == dt and y.shape == x.shape
    assert ((y.double() - want).abs() <= want.abs() * (_u(dt) + TINY) + torch.finfo(dt).tiny).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,D", [(1, 32), (3, 96), (8, 1024), (5, 2080), (3, 4096), (2, 8192), (2, 9216 - 32), (1, 32800)])
def test_mxfp8(dev, dt, T, D):
    from lockstep_amd.norm import add_rms_norm
    dt = DT[dt]
    x, r, w = _inputs(dev, T, D, dt, D + T)
    y, h, codes, scale = add_rms_norm(x, w, r, mxfp8=True)
    want, _ = _exact(h, w, 1e-6)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scale.shape == (T, D // 32)
    _check_mx8(codes, scale, want)
    y2, codes2, scale2 = add_rms_norm(h, w, mxfp8=True)
    assert torch.equal(y2, y) and torch.equal(codes2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scale2, scale)
    assert torch.equal(y, add_rms_norm(x, w, r)[0])


def test_mxfp8_of_zeros_infinities_and_small_values(dev):
    from lockstep_amd.norm import add_rms_norm
    x = torch.zeros((4, 96), device=dev)
    w = torch.ones(96, device=dev)
    x[1, 5] = float("nan")                    # spreads over the row, as it does in the formula
    w2 = w.clone()
    w2[40] = float("inf")                     # one block of every row
    x[2] = 1.0
    x[3, 64:] = 2.0 ** -140                   # below the least normal number, beside ones
    x[3, :64] = 1.0
    y, codes, scale = add_rms_norm(x, w, mxfp8=True)
    assert (scale[0] == 127).all() and (codes[0].float() == 0).all() and (y[0] == 0).all()
    assert (scale[1] == 255).all() and torch.isnan(y[1]).all()
    assert (scale[2] == 127 - 8).all()
    assert (scale[3, 2] == 0) and torch.isfinite(codes[3].float()).all()
    y, codes, scale = add_rms_norm(x[2:3], w2, mxfp8=True)
    assert scale[0].tolist() == [119, 255, 119] and torch.isinf(y[0, 40])


def test_least_scale_at_the_border(dev):
    """A block whose largest is 448 * 2^e keeps scale 2^e; one step more takes the next."""
    from lockstep_amd.norm import add_rms_norm
    x = torch.ones((1, 64), device=dev)       # norm 1 with eps 0: y = w
    w = torch.ones(64, device=dev)
    w[3] = 448.0
    w[40] = 448.0 + 2.0 ** -15
    _, codes, scale = add_rms_norm(x, w, eps=0.0, mxfp8=True)
    assert scale[0].tolist() == [127, 128]
    assert codes[0, 3].float() == 448 and codes[0, 40].float() == 224 and codes[0, 0].float() == 1


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,D", [(1, 1), (3, 7), (1500, 64), (70, 520), (33, 2048), (5, 2051), (1030, 96), (9, 4096), (3, 8192),
                                 (2, 8200), (3, 9001)])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients(dev, dt, T, D, residual):
    from lockstep_amd.norm import add_rms_norm
    dt = DT[dt]
    x, r, w = _inputs(dev, T, D, dt, 3 * D + T, torch.float32 if T % 2 else None)
    g = torch.Generator(device=dev).manual_seed(T)
    dy, dh = (torch.randn((T, D), generator=g, device=dev).to(dt) for _ in range(2))
    leaves = [t.requires_grad_(True) for t in ((x, w, r) if residual else (x, w))]
    got = add_rms_norm(x, w, r if residual else None)
    outs, up = (got, (dy, dh)) if residual else ((got,), (dy,))
    grads = torch.autograd.grad(outs, leaves, up)
    h = got[1].detach() if residual else x.detach()
    _, inv = _exact(h, w, 1e-6)
    gw, hd, dyd = dy.double() * w.detach().double(), h.double(), dy.double()
    mean = (gw * hd).mean(-1, keepdim=True)
    want = inv * (gw - hd * inv ** 2 * mean) + (dh.double() if residual else 0)
    mag = inv * (gw.abs() + hd.abs() * inv ** 2 * (gw * hd).abs().mean(-1, keepdim=True)) + (dh.double().abs() if residual else 0)
    assert ((grads[0].double() - want).abs() <= want.abs() * _u(dt) + mag * TINY + torch.finfo(dt).tiny).all()
    if residual:
        assert torch.equal(grads[2], grads[0])
    dw, mag = (dyd * hd * inv).sum(0), (dyd * hd * inv).abs().sum(0)
    assert grads[1].dtype == w.dtype
    assert ((grads[1].double() - dw).abs() <= dw.abs() * _u(w.dtype) + mag * TINY + torch.finfo(w.dtype).tiny).all()
    again = torch.autograd.grad(add_rms_norm(x, w, r if residual else None), leaves, up)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_gradient_against_differences(dev):
    from lockstep_amd.norm import add_rms_norm
    g = torch.Generator(device=dev).manual_seed(0)
    x, r, w = (torch.randn(s, generator=g, device=dev) for s in ((2, 24), (2, 24), (24,)))
    cy, ch = (torch.randn((2, 24), generator=g, device=dev).double() for _ in range(2))

    def loss(*t):
        y, h = add_rms_norm(*t)
        return float((y.double() * cy).sum() + (h.double() * ch).sum())
    leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, h = add_rms_norm(*leaves)
    grads = torch.autograd.grad((y, h), leaves, (cy.float(), ch.float()))
    for i, t in enumerate((x, w, r)):
        for at in (0, 5, t.numel() - 1):
            step = torch.zeros_like(t)
            step.view(-1)[at] = 2.0 ** -7
            args = [x, w, r]
            up, down = list(args), list(args)
            up[i], down[i] = t + step, t - step
            # differences: second-order error of step^2, rounding of 2^-23 over the step
            assert abs((loss(*up) - loss(*down)) / 2.0 ** -6 - float(grads[i].view(-1)[at])) < 5e-3


def test_partial_gradients(dev):
    """Only some of the inputs, only some of the outputs, and no rows."""
    from lockstep_amd.norm import add_rms_norm
    x, r, w = _inputs(dev, 4, 64, torch.float32, 1)
    xg = x.clone().requires_grad_(True)
    y, h = add_rms_norm(xg, w, r)
    full, = torch.autograd.grad(y.sum() + h.sum(), xg, retain_graph=True)
    only_h, = torch.autograd.grad(h.sum(), xg, retain_graph=True)
    only_y, = torch.autograd.grad(y.sum(), xg)
    assert torch.equal(only_h, torch.ones_like(x))
    assert (full - only_h - only_y).abs().max() <= 2.0 ** -20 * (1 + only_y.abs().max())
    wg = w.clone().requires_grad_(True)
    y, h = add_rms_norm(x, wg, r)
    y.sum().backward()
    assert wg.grad is not None
    e = torch.zeros((0, 64), device=dev, requires_grad=True)
    wg.grad = None
    add_rms_norm(e, wg).sum().backward()
    assert e.grad.shape == (0, 64) and torch.equal(wg.grad, torch.zeros_like(w))


def test_strides_shapes_and_placement(dev):
    """Any strides and leading shape, rows that are not aligned, an expanded
    residual: the same results as contiguous ones."""
    from lockstep_amd.norm import add_rms_norm
    g = torch.Generator(device=dev).manual_seed(2)
    base = torch.randn((3, 5, 2 * 96 + 2), generator=g, device=dev).bfloat16()
    w = torch.randn(96, generator=g, device=dev).bfloat16()
    for x in (base[..., :96], base[..., 1:97], base[..., :192:2], base[:, :, 2:98].transpose(0, 1), base[:1, :1, :96]):
        r = torch.ones((), device=dev, dtype=torch.bfloat16).expand(x.shape)
        got, want = add_rms_norm(x, w, r, mxfp8=True), add_rms_norm(x.contiguous(), w, r.contiguous(), mxfp8=True)
        for p, q in zip(got, want):
            assert p.shape == q.shape and torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))
        a, b = x.detach().clone().requires_grad_(True), x.detach().requires_grad_(True)
        dy = torch.randn((*x.shape[:-1], 97), generator=g, device=dev).bfloat16()[..., 1:]
        p, = torch.autograd.grad(add_rms_norm(a.contiguous(), w), a, dy.contiguous())
        q, = torch.autograd.grad(add_rms_norm(b, w), b, dy)
        assert torch.equal(p, q)
    one = torch.randn(40, generator=g, device=dev)
    assert add_rms_norm(one, torch.ones(40, device=dev)).shape == (40,)
    assert add_rms_norm(base[:0, :, :96], w, mxfp8=True)[1].shape == (0, 5, 96)


def test_on_another_stream_and_replayed(dev):
    from lockstep_amd.norm import add_rms_norm
    x, r, w = _inputs(dev, 40, 4096, torch.bfloat16, 5)
    want = add_rms_norm(x, w, r, mxfp8=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = add_rms_norm(x, w, r, mxfp8=True)
    s.synchronize()
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = add_rms_norm(x, w, r, mxfp8=True)
    for k in range(3):
        x.normal_(generator=torch.Generator(device=dev).manual_seed(k))
        graph.replay()
        torch.cuda.synchronize()
        want = add_rms_norm(x, w, r, mxfp8=True)
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(out, want))


def test_feeds_the_fp8_product(dev):
    """The codes and scales are operands of mxfp4_gemm_fp8: MXFP8 rows times MXFP4 weights."""
    from lockstep_amd import fp4, mxfp4_gemm
    from lockstep_amd.norm import add_rms_norm
    x, r, w = _inputs(dev, 96, 256, torch.bfloat16, 9)
    g = torch.Generator(device=dev).manual_seed(4)
    codes, scale = fp4.quantize_mxfp4(torch.randn((128, 256), generator=g, device=dev))
    _, _, x8, xs = add_rms_norm(x, w, r, mxfp8=True)
    we = (scale.view(torch.int32) >> 23).to(torch.uint8)
    got = mxfp4_gemm.mxfp4_gemm_fp8(x8, fp4.codes_to_e4m3(codes).t().contiguous(), xs, we.t().contiguous(), out_dtype=torch.float32)
    xv = x8.double() * torch.exp2(xs.double() - 127).repeat_interleave(32, 1)
    wv = fp4.dequantize_mxfp4(codes, scale).double()
    mag = xv.abs() @ wv.abs().t()
    assert ((got.double() - xv @ wv.t()).abs() <= mag * 2.0 ** -12).all()

"""Sink-window attention against the formula in 64 bits, forward and gradients.

Tolerances.  Scores and sums are fp32; what is rounded to u = 2^-9 (bf16) or
2^-12 (fp16, half an ulp of 1) relative is each probability (and dS) once, the
output o once (which enters delta), and each result once.  An output is a
p-weighted mean of |v| <= V: |err| <= (u + u) max|v| + fp32 noise; gradients are
sums of n terms of magnitude t: the rounding of the terms gives at most
u sum|t|, and that of o at most u |o| |dO| in delta, bounded together by
4 u (sum |t|) with the result's own rounding.  The sums of magnitudes are
computed in 64 bits beside the results, so the bound is per element."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # one rounding, at most half of this


def visible(tq, tk, window, sinks, dev):
    p = torch.arange(tq, device=dev)[:, None] + tk - tq
    j = torch.arange(tk, device=dev)[None]
    see = j <= p
    if window is not None:
        see = see & ((j > p - window) | (j < sinks))
    return see


def formula(q, k, v, window, sinks, scale, do=None):
    """One sequence [T, H, D] in float64: o, lse, gradients, and the sums of
    magnitudes that bound each one's rounding."""
    G = q.shape[1] // k.shape[1]
    q, k, v = q.double().transpose(0, 1), k.double().transpose(0, 1), v.double().transpose(0, 1)
    kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    see = visible(q.shape[1], k.shape[1], window, sinks, q.device)
    s = torch.where(see, scale * (q @ kk.transpose(1, 2)), -math.inf)
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:2], 1), -math.inf)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m)) * see
    tot = e.sum(-1, keepdim=True)
    p = e / torch.where(tot == 0, 1.0, tot)
    o = p @ vv
    lse = torch.where(tot == 0, -math.inf, m + torch.log(tot))[..., 0]
    got = {"o": o.transpose(0, 1), "lse": lse, "o_mag": (p @ vv.abs()).transpose(0, 1)}
    if do is not None:
        do = do.double().transpose(0, 1)
        dp = do @ vv.transpose(1, 2)
        delta = (do * o).sum(-1, keepdim=True)
        delta_mag = (do.abs() * o.abs()).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        ds_mag = p * ((dp - delta).abs() + delta_mag)
        fold = lambda x: x.unflatten(0, (-1, G)).sum(1).transpose(0, 1)  # noqa: E731
        got.update(dq=scale * (ds @ kk).transpose(0, 1), dk=fold(scale * (ds.transpose(1, 2) @ q)),
                   dv=fold(p.transpose(1, 2) @ do))
        got.update(dq_mag=scale * (ds_mag @ kk.abs()).transpose(0, 1),
                   dk_mag=fold(scale * (ds_mag.transpose(1, 2) @ q.abs())), dv_mag=fold(p.transpose(1, 2) @ do.abs()))
    return got


def close(name, x, ref, mag, u, n):
    assert torch.isfinite(x).all(), name
    tol = 4 * u * mag + 1e-6 * mag + 2e-6 * n
    bad = (x.double() - ref).abs() - tol
    assert bad.max().item() <= 0, f"{name}: {bad.max().item():.3e} over the bound at {bad.argmax().item()}"


def inputs(B, Tq, Tk, H, Hkv, D, dt, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=dev).to(dt)  # noqa: E731
    return r(B, Tq, H, D), r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), r(B, Tq, H, D)


CASES = [
    # B, Tq, Tk, H, Hkv, D, window, sinks
    (1, 1, 1, 1, 1, 8, None, 0),
    (2, 1, 77, 4, 2, 64, None, 0),
    (2, 63, 63, 3, 3, 64, None, 0),
    (1, 65, 65, 6, 2, 128, 16, 1),
    (2, 200, 200, 4, 1, 72, 1, 0),        # sees itself alone
    (1, 300, 300, 2, 2, 128, 33, 70),     # sinks over more than one tile
    (1, 129, 500, 8, 2, 128, 100, 4),     # keys before the queries
    (2, 150, 40, 5, 1, 64, None, 0),      # 110 rows see nothing
    (1, 700, 700, 10, 2, 96, 257, 5),
    (3, 256, 256, 4, 4, 128, 5000, 3),    # a window longer than the sequence
    (1, 515, 515, 7, 1, 40, 64, 64),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case, dt, dev):
    from lockstep_amd.attention import sink_window_attention
    B, Tq, Tk, H, Hkv, D, window, sinks = case
    q, k, v, do = inputs(B, Tq, Tk, H, Hkv, D, dt, dev, seed=Tq)
    scale = 1.0 / math.sqrt(D)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    o, lse = sink_window_attention(q, k, v, window=window, sinks=sinks, return_lse=True)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    for b in range(B):
        ref = formula(q[b].detach(), k[b].detach(), v[b].detach(), window, sinks, scale, do[b])
        close("o", o[b].detach(), ref["o"], ref["o_mag"], U[dt], 1)
        fin = torch.isfinite(ref["lse"])
        assert torch.equal(fin, torch.isfinite(lse[b])) and (lse[b][~fin] == -math.inf).all()
        assert ((lse[b].double() - ref["lse"])[fin].abs() <= 1e-5 * (1 + ref["lse"][fin].abs())).all()
        for n, x in (("dq", dq), ("dk", dk), ("dv", dv)):
            close(n, x[b], ref[n], ref[n + "_mag"], U[dt], 1)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[1], [5, 0, 130, 64], [300, 1, 1, 257], [0, 0], list(range(1, 70))])
def test_packed_sequences(lens, dt, dev):
    from lockstep_amd.attention import sink_window_attention
    head, tail = 3, 9                       # tokens that belong to no sequence
    N, H, Hkv, D = head + sum(lens) + tail, 4, 2, 64
    q, k, v, do = (t[0] for t in inputs(1, N, N, H, Hkv, D, dt, dev, seed=len(lens)))
    off = [head + sum(lens[:b]) for b in range(len(lens) + 1)]
    offsets = torch.tensor(off, dtype=torch.int32, device=dev)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    o, lse = sink_window_attention(q, k, v, window=50, sinks=2, offsets=offsets, return_lse=True)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    for lo, hi in zip(off, off[1:]):
        if hi == lo:
            continue
        ref = formula(*(t[lo:hi].detach() for t in (q, k, v)), 50, 2, 1.0 / math.sqrt(D), do[lo:hi])
        close("o", o[lo:hi].detach(), ref["o"], ref["o_mag"], U[dt], 1)
        assert ((lse[:, lo:hi].double() - ref["lse"]).abs() <= 1e-5 * (1 + ref["lse"].abs())).all()
        for n, x in (("dq", dq), ("dk", dk), ("dv", dv)):
            close(n, x[lo:hi], ref[n], ref[n + "_mag"], U[dt], 1)
    for sl in (slice(0, head), slice(off[-1], N)):
        for t in (o, dq, dk, dv):
            assert (t[sl] == 0).all()
        assert (lse[:, sl] == -math.inf).all()


def test_strided_and_broadcast_inputs(dev):
    """Views of one fused projection, a head broadcast over all, offset bases."""
    from lockstep_amd.attention import sink_window_attention
    g = torch.Generator(device=dev).manual_seed(5)
    qkv = torch.randn((2, 90, 8, 3, 64), generator=g, device=dev).bfloat16()
    q, k, v = qkv[:, :, :, 0], qkv[:, :, :4, 1], qkv[:, :, :4, 2]
    want = sink_window_attention(q.contiguous(), k.contiguous(), v.contiguous(), window=20, sinks=3)
    assert torch.equal(sink_window_attention(q, k, v, window=20, sinks=3), want)
    odd = torch.randn((2, 90, 8, 67), generator=g, device=dev).bfloat16()   # rows of 134 bytes
    x = odd[..., 3:]
    assert torch.equal(sink_window_attention(x, k, v), sink_window_attention(x.clone(), k, v))
    one = torch.randn((2, 90, 1, 64), generator=g, device=dev).bfloat16().requires_grad_(True)
    o = sink_window_attention(q, one.expand(-1, -1, 4, -1), v)
    d1, = torch.autograd.grad(o, one, torch.ones_like(o))
    o = sink_window_attention(q, one.repeat(1, 1, 4, 1), v)
    d2, = torch.autograd.grad(o, one, torch.ones_like(o))
    assert torch.equal(d1, d2)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)                      # heads outside tokens
    assert torch.equal(sink_window_attention(t, k, v, window=20, sinks=3), want)


def test_gradients_against_differences(dev):
    """The loss sum(o w) along random directions, in the kernels' own forward:
    a central difference of step h has error O(h^2) plus the outputs' rounding
    over h, both far below the tolerance of 2%."""
    from lockstep_amd.attention import sink_window_attention
    q, k, v, w = inputs(1, 150, 150, 4, 2, 64, torch.float16, dev, seed=3)
    xs = [t.float().requires_grad_(True) for t in (q, k, v)]
    o = sink_window_attention(*(t.half() for t in xs), window=40, sinks=2)
    grads = torch.autograd.grad((o.float() * w.float()).sum(), xs)
    g = torch.Generator(device=dev).manual_seed(9)
    for i, gr in enumerate(grads):
        d = torch.sign(torch.randn(gr.shape, generator=g, device=dev)) * torch.sign(gr)  # half along the gradient
        d = torch.where(torch.rand(gr.shape, generator=g, device=dev) < 0.5, torch.sign(gr), d)
        h = 2.0 ** -6
        f = []
        for s in (h, -h):
            y = [t.detach() for t in xs]
            y[i] = (y[i] + s * d).half().float()
            step = y[i] - xs[i].detach()
            f.append(((sink_window_attention(*(t.half() for t in y), window=40, sinks=2).double() * w.double()).sum(),
                      (step.double() * gr.double()).sum()))
        num, lin = f[0][0] - f[1][0], f[0][1] - f[1][1]
        assert abs(num - lin) <= 0.02 * abs(lin), (i, num.item(), lin.item())


def test_deterministic_and_on_another_stream(dev):
    from lockstep_amd.attention import sink_window_attention
    q, k, v, do = inputs(2, 400, 400, 8, 2, 128, torch.bfloat16, dev, seed=1)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    def once():
        o = sink_window_attention(q, k, v, window=100, sinks=4)
        return (o, *torch.autograd.grad(o, (q, k, v), do))
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = once()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_empty_and_refused(dev):
    from lockstep_amd.attention import sink_window_attention as f
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=dev)  # noqa: E731
    assert f(z(0, 4, 2, 64), z(0, 4, 2, 64), z(0, 4, 2, 64)).shape == (0, 4, 2, 64)
    assert f(z(2, 0, 2, 64), z(2, 5, 2, 64), z(2, 5, 2, 64)).shape == (2, 0, 2, 64)
    assert (f(z(2, 3, 2, 64) + 1, z(2, 0, 2, 64), z(2, 0, 2, 64)) == 0).all()
    q = z(2, 0, 2, 64).requires_grad_(True)
    k = z(2, 5, 2, 64).requires_grad_(True)
    o = f(q, k, k.detach())
    assert (torch.autograd.grad(o.sum(), k)[0] == 0).all()
    q, k = z(1, 4, 4, 64), z(1, 4, 2, 64)
    with pytest.raises(TypeError):
        f(q.float(), k.float(), k.float())
    with pytest.raises(TypeError):
        f(q, k.half(), k)
    with pytest.raises(AssertionError):
        f(q, z(1, 4, 3, 64), z(1, 4, 3, 64))
    with pytest.raises(AssertionError):
        f(z(1, 4, 4, 136), z(1, 4, 4, 136), z(1, 4, 4, 136))
    with pytest.raises(AssertionError):
        f(z(1, 4, 4, 12), z(1, 4, 4, 12), z(1, 4, 4, 12))
    with pytest.raises(AssertionError):
        f(q, k, z(1, 5, 2, 64))
    with pytest.raises(AssertionError):
        f(q[0], k[0], k[0])
    with pytest.raises(AssertionError):
        f(q[0], k[0], k[0], offsets=torch.tensor([0, 4], device=dev))
    for bad in ({"window": 0}, {"sinks": -1}, {"scale": 0.0}, {"scale": float("inf")}, {"scale": float("nan")}):
        with pytest.raises(ValueError):
            f(q, k, k, **bad)
    with pytest.raises(RuntimeError):
        f(q.cpu(), k.cpu(), k.cpu())

"""Attention and cache: each launch form, the native calls against the Python
ones, values at the ends of their types, and a layer that runs them together.
Tolerances as in test_gpu_attention.py and test_gpu_kv_cache.py; where one
differs its test derives it."""

import math

import pytest
import torch

from .test_gpu_attention import U, close, formula, inputs
from .test_gpu_kv_cache import filled, held, reference_evict
from .test_gpu_kv_cache import formula as cache_formula

pytestmark = pytest.mark.gpu


@pytest.fixture
def python_calls(monkeypatch):
    """Without the native call path."""
    from lockstep_amd import _capi

    class Nothing:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(_capi, "fast", Nothing())


# waves of 16 rows: 1600 (keys in halves), 2550 (16 rows a wave), 4250 (32 rows
# at head 128), 6800 (32 at head 64)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,D,window,sinks", [(2, 800, 64, None, 0), (3, 850, 64, 200, 3), (8, 850, 64, 200, 3),
                                                (2, 800, 128, 200, 3), (3, 850, 128, None, 0), (5, 850, 128, 200, 70)])
def test_forms(B, T, D, window, sinks, dt, dev):
    from lockstep_amd.attention import sink_window_attention
    H, Hkv = 16, 4
    q, k, v, do = inputs(B, T, T, H, Hkv, D, dt, dev, seed=B)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    o = sink_window_attention(q, k, v, window=window, sinks=sinks)
    grads = torch.autograd.grad(o, (q, k, v), do)
    for b in (0, B - 1):
        ref = formula(q[b].detach(), k[b].detach(), v[b].detach(), window, sinks, 1.0 / math.sqrt(D), do[b])
        close("o", o[b].detach(), ref["o"], ref["o_mag"], U[dt], 1)
        for n, x in zip(("dq", "dk", "dv"), grads):
            close(n, x[b], ref[n], ref[n + "_mag"], U[dt], 1)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,D,window,sinks", [(3, 850, 64, 200, 3), (8, 850, 64, 200, 3), (3, 850, 128, None, 0),
                                                (5, 850, 128, 200, 70)])
def test_cache_forms(B, T, D, window, sinks, dt, dev):
    from lockstep_amd import kv_cache as kc
    H, Hkv, lens = 16, 4, [850 + 13 * b for b in range(B)]
    pages, table, lengths, (kv, vv), _ = filled(lens, Hkv, D, 32, dt, dev, seed=T + D)
    q = inputs(B, T, 1, H, Hkv, D, dt, dev, seed=3)[0]
    w = torch.zeros((B, Hkv, table.shape[1] * 32), device=dev)
    o = kc.attend(q, pages, table, lengths, window=window, sinks=sinks, weights=w)
    for b in (0, B - 1):
        ro, mag, rw, err = cache_formula(q[b], kv[b], vv[b], window, sinks, 1.0 / math.sqrt(D))
        assert ((o[b].double() - ro).abs() <= 4 * U[dt] * mag + 1e-7).all()
        bad = (w[b, :, :lens[b]].double() - rw).abs() - err - 2.0 ** -22 * rw
        assert bad.max().item() <= 0, bad.max().item()
        assert (w[b, :, lens[b]:] == 0).all()


@pytest.mark.parametrize("n,keep", [(9001, 4000), (40000, 20001), (33001, 1)])
def test_evict_long(n, keep, dev):
    """More positions than a workgroup holds in registers."""
    from lockstep_amd import kv_cache as kc
    page = 256
    g = torch.Generator(device=dev).manual_seed(n)
    count, more = -(-n // page), -(-keep // page)
    pages = kc.new_pages(count + more, 1, 64, page, device=dev)
    for t in pages:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=dev, dtype=torch.uint8))
    table = torch.randperm(count, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None].to(dev)
    out = torch.arange(count, count + more, dtype=torch.int32, device=dev)[None]
    lengths = torch.tensor([n], dtype=torch.int32, device=dev)
    w = torch.randint(0, 50, (1, 1, count * page), generator=g, device=dev).float() / 7
    before = [t.clone() for t in pages]
    index, kept, new = kc.evict(pages, table, lengths, w, keep, out, sinks=min(4, keep - 1), recent=0)
    want = reference_evict(w[0, 0].tolist(), n, keep, min(4, keep - 1), 0)
    assert new.item() == keep and index[0, 0].tolist() == want
    at = torch.tensor(want, device=dev)
    assert torch.equal(kept[0, 0], w[0, 0, at])
    for s, d in zip(held(before, table, 0, n, page, dev), held(pages, out, 0, keep, page, dev)):
        assert torch.equal(s[at], d)


def test_native_and_python_calls_agree(dev, request):
    from lockstep_amd import kv_cache as kc
    from lockstep_amd.attention import sink_window_attention as f
    q, k, v, do = inputs(2, 90, 90, 6, 2, 64, torch.bfloat16, dev, seed=5)
    packed = [torch.randn((100, 3, h, 64), device=dev, generator=torch.Generator(device=dev).manual_seed(h)).half()[:, 1]
              for h in (4, 2, 2)]
    off = torch.tensor([0, 30, 30, 95], dtype=torch.int32, device=dev)
    pages, table, lengths, _, (kn, vn) = filled([70, 33], 2, 64, 16, torch.bfloat16, dev, seed=2)
    w0 = torch.rand((2, 2, table.shape[1] * 16), generator=torch.Generator(device=dev).manual_seed(1), device=dev)

    def run():
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = f(*x, window=20, sinks=1, scale=0.2)
        got = [o, *torch.autograd.grad(o, x, do), f(q, k, v), f(*packed, offsets=off, window=9)]
        y = [t.clone().requires_grad_(True) for t in packed]
        o = f(*y, offsets=off, sinks=3, window=5)
        got += [o, *torch.autograd.grad(o.square().sum(), y)]
        p = kc.Pages(*(t.clone() for t in pages))
        got += kc.append(p, kn.view(1, -1, 2, 64)[:, :66].reshape(2, 33, 2, 64), vn.view(1, -1, 2, 64)[:, :66].reshape(2, 33, 2, 64),
                         table, lengths, values=True)
        kc.append(p, kn, vn, table, lengths, offsets=torch.tensor([0, 70, 103], dtype=torch.int32, device=dev))
        w = w0.clone()
        got += [kc.attend(q[:, :1], p, table, lengths, weights=w), kc.attend(q[:, :80], p, table, lengths, window=11, sinks=2), w]
        p = kc.Pages(*(torch.cat([t, torch.zeros_like(t)]) for t in p))
        got += kc.evict(p, table, lengths, w, 20, torch.tensor([[20, 21], [22, 23]], dtype=torch.int32, device=dev), recent=3)
        return [t.detach() for t in got] + list(p)
    native = run()
    request.getfixturevalue("python_calls")
    for i, (a, b) in enumerate(zip(native, run(), strict=True)):
        assert a.dtype == b.dtype and torch.equal(a, b), i


def test_hidden_values_do_not_matter(dev):
    """NaN in other sequences, in tokens of none, and in keys that no row of
    the result sees, forward and backward."""
    from lockstep_amd.attention import sink_window_attention as f
    N, off = 400, [10, 140, 300]
    offsets = torch.tensor(off, dtype=torch.int32, device=dev)
    q, k, v, do = (t[0] for t in inputs(1, N, N, 4, 2, 128, torch.bfloat16, dev, seed=8))
    def run(*x):
        x = [t.clone().requires_grad_(True) for t in x]
        o = f(*x, offsets=offsets, window=40, sinks=2)
        return (o.detach(), *torch.autograd.grad(o, x, d))
    d = do
    clean = run(q, k, v)
    bad = [t.clone() for t in (q, k, v, do)]
    for t in bad:
        t[:10], t[140:] = math.nan, math.inf
    d = bad[3]
    for a, b in zip(clean, run(*bad[:3])):
        assert torch.equal(a[10:140], b[10:140])
        assert (b[:10] == 0).all() and (b[300:] == 0).all()
    # a NaN key hides from the rows before it, and from those past its window
    k2 = k.clone()
    k2[200] = math.nan
    o = f(q, k2, v, offsets=offsets, window=40, sinks=2)
    assert torch.equal(o[140:200], clean[0][140:200]) and torch.equal(o[240:300], clean[0][240:300])
    assert torch.isnan(o[200:240]).all()


def test_fp16_gradients_at_the_ends_of_the_type(dev):
    """Small and large dO in one call: every result is within the bound of its
    own magnitude, and fp16's spacing near zero (2^-24, half of it rounding)."""
    from lockstep_amd.attention import sink_window_attention as f
    q, k, v, do = inputs(1, 300, 300, 4, 2, 64, torch.float16, dev, seed=6)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    for lo, hi in ((-14, -14), (-20, -12), (-16, 4), (6, 6)):
        e = torch.linspace(lo, hi, 300, device=dev).round()
        d = (do.float() * torch.exp2(e)[None, :, None, None]).half()
        grads = torch.autograd.grad(f(*x, window=100, sinks=2), x, d)
        ref = formula(q[0].detach(), k[0].detach(), v[0].detach(), 100, 2, 0.125, d[0])
        for n, g in zip(("dq", "dk", "dv"), grads):
            assert torch.isfinite(g).all()
            bad = (g[0].double() - ref[n]).abs() - 4 * U[torch.float16] * ref[n + "_mag"] - 2.0 ** -24
            assert bad.max().item() <= 0, (lo, hi, n, bad.max().item())


def test_large_scores(dev):
    """Scores of thousands: one key takes all, the others' weights are 0."""
    from lockstep_amd.attention import sink_window_attention as f
    q, k, v, _ = inputs(1, 200, 200, 2, 2, 64, torch.bfloat16, dev, seed=9)
    q, k = q * 16, k * 16
    o, lse = f(q, k, v, return_lse=True)
    ref = formula(q[0], k[0], v[0], None, 0, 0.125)
    assert torch.isfinite(o).all()
    # a score s has an absolute error of 2^-20 (|s| terms): of the weights, that
    # much relative; the terms' sum is at most 0.125 sum |q k| < 2^13 here
    err = 2.0 ** -20 * 0.125 * (q[0].double().abs().transpose(0, 1) @ k[0].double().abs().permute(1, 2, 0)).amax()
    assert ((o[0].double() - ref["o"]).abs() <= (4 * U[torch.bfloat16] + 2 * err) * v.abs().max().item()).all()
    assert ((lse[0].double() - ref["lse"]).abs() <= err + 1e-5 * ref["lse"].abs()).all()


def test_autocast_and_second_derivatives(dev):
    from lockstep_amd.attention import sink_window_attention as f
    q, k, v, do = inputs(1, 40, 40, 2, 1, 64, torch.bfloat16, dev, seed=4)
    x = [t.float().requires_grad_(True) for t in (q, k, v)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        o = f(*x)
    assert o.dtype == torch.bfloat16 and torch.equal(o, f(q, k, v))
    grads = torch.autograd.grad(o, x, do)
    assert all(g.dtype == torch.float32 for g in grads)
    y = [t.requires_grad_(True) for t in (q, k, v)]
    for a, b in zip(grads, torch.autograd.grad(f(*y), y, do)):
        assert torch.equal(a, b.float())
    first = torch.autograd.grad(f(*y).float().square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first[0].float().sum(), y[1], retain_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first[0].float().sum().backward()


# --------------------------------------------------------------- the layer

def layer_of(dev, **kw):
    from lockstep_amd.fp4_attention import MXFP4SelfAttention
    torch.manual_seed(0)
    return MXFP4SelfAttention(512, 8, 2, **kw).to(dev, torch.bfloat16)


def test_layer_gradients(dev):
    """dX of the layer: the linears' backward is unquantized, so it is
    [dq dk dv] Wqkv with the attention's gradients for dO = G Wout.  Each of
    dO and [dq dk dv] is rounded to bf16 once more on the way: 2^-9 of the
    magnitudes, within the bound's 4 u with the u added here."""
    layer = layer_of(dev, window=48, sinks=2)
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((2, 128, 512), generator=g, device=dev).bfloat16().requires_grad_(True)
    gy = torch.randn((2, 128, 512), generator=g, device=dev).bfloat16()
    layer(x).backward(gy)
    q, k, v = (t.detach() for t in layer._split(layer.qkv(x)))
    w = layer.qkv.weight.detach().double()
    for b in range(2):
        do = (gy[b] @ layer.out.weight.detach()).unflatten(-1, (8, 64))
        ref = formula(q[b], k[b], v[b], 48, 2, 0.125, do)
        cat = lambda s: torch.cat([ref["d" + n + s].flatten(1) for n in "qkv"], 1)  # noqa: E731
        want, mag = cat("") @ w, cat("_mag") @ w.abs()
        assert ((x.grad[b].double() - want).abs() <= 5 * U[torch.bfloat16] * mag + 1e-6).all()
    assert all(torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in layer.parameters())


def test_layer_served(dev):
    """Prompts, single tokens, a chunk and an eviction; Wout is the identity,
    exact in MXFP4, so that the outputs are the attention's."""
    from lockstep_amd.mxfp4_gemm import mxfp4_linear_w
    from lockstep_amd import fp4
    layer = layer_of(dev, window=None, sinks=2)
    with torch.no_grad():
        layer.out.weight.copy_(torch.eye(512))
    layer.pack()
    cache = layer.new_cache(2, 256, page_size=16, track=True)
    g = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device=dev).bfloat16()  # noqa: E731
    offsets = torch.tensor([0, 70, 100], dtype=torch.int32, device=dev)
    x = r(100, 512)
    y = layer.prefill(x, cache, offsets, longest=70)
    q, k, v = layer._split(mxfp4_linear_w(x, *layer.packed[0]))
    for lo, hi in ((0, 70), (70, 100)):
        ref = formula(q[lo:hi], k[lo:hi], v[lo:hi], None, 0, 0.125)
        close("prefill", y[lo:hi].unflatten(-1, (8, 64)), ref["o"], ref["o_mag"], U[torch.bfloat16], 1)
    assert cache.lengths.tolist() == [70, 30] and cache.used == 70

    def check(T):
        x = r(2, T, 512)
        w0 = cache.weights.clone()
        y = layer.step(x, cache).unflatten(-1, (8, 64))
        q = layer._split(mxfp4_linear_w(x, *layer.packed[0]))[0]
        for b, n in enumerate(cache.lengths.tolist()):
            kc_, ks, vc, vs = held(cache.pages, cache.table, b, n, 16, dev)
            k, v = (fp4.dequantize_packed(c.contiguous().flatten(0, 1), s.contiguous().flatten(0, 1)).view(n, 2, 64)
                    for c, s in ((kc_, ks), (vc, vs)))
            ro, mag, rw, err = cache_formula(q[b], k, v, None, 0, 0.125)
            assert ((y[b].double() - ro).abs() <= 4 * U[torch.bfloat16] * mag + 1e-7).all()
            new = w0[b, :, :n].double() + rw
            assert ((cache.weights[b, :, :n].double() - new).abs() <= err + 2.0 ** -22 * new).all()
    for T in (1, 1, 70, 1):
        check(T)
    index = cache.evict(64, recent=16)
    assert cache.lengths.tolist() == [64, 64] and cache.used == 64 and index.shape == (2, 2, 64)
    assert (index[:, :, :2] == torch.arange(2, device=dev)).all()
    for T in (1, 5):
        check(T)
    with pytest.raises(ValueError, match="holds 256"):
        layer.step(r(2, 200, 512), cache)
    with pytest.raises(ValueError, match="empty cache"):
        layer.prefill(x, cache, offsets)
    with pytest.raises(ValueError, match="track"):
        layer.new_cache(1, 16, page_size=16).evict(4)
    with pytest.raises(RuntimeError, match="pack"):
        layer_of(dev).step(r(2, 1, 512), cache)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,D,window", [(2, 8, 64, None), (3, 12, 128, 300), (2, 17, 64, 500), (20, 30, 64, None),
                                          (18, 45, 128, 900), (20, 52, 64, None), (18, 60, 128, None)])
def test_cache_weights_of_some_rows(B, T, D, window, dt, dev):
    """32 to 240 rows of a key head over few and many keys: each form of the
    weights' pass, and the shares of attention's."""
    from lockstep_amd import kv_cache as kc
    H, Hkv, lens = 8, 2, [1000 - 7 * b for b in range(B)]
    pages, table, lengths, (kv, vv), _ = filled(lens, Hkv, D, 64, dt, dev, seed=T)
    q = inputs(B, T, 1, H, Hkv, D, dt, dev, seed=7)[0]
    w0 = torch.rand((B, Hkv, table.shape[1] * 64), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    w = w0.clone()
    o = kc.attend(q, pages, table, lengths, window=window, sinks=3, weights=w)
    for b in (0, B - 1):
        ro, mag, rw, err = cache_formula(q[b], kv[b], vv[b], window, 3, 1.0 / math.sqrt(D))
        bad = (o[b].double() - ro).abs() - 4 * U[dt] * mag - 1e-7
        assert bad.max().item() <= 0, bad.max().item()
        new = w0[b].double()
        new[:, :lens[b]] += rw
        tol = 2.0 ** -22 * new
        tol[:, :lens[b]] += err
        bad = (w[b].double() - new).abs() - tol
        assert bad.max().item() <= 0, bad.max().item()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hkv,D,window,sinks", [
    (1, 1500, 1500, 5, 1, 64, None, 0),      # few key tiles, long and short
    (1, 700, 1300, 6, 2, 128, None, 0),      # keys before the queries
    (1, 1300, 700, 4, 1, 80, None, 3),       # rows that see nothing
    (2, 1100, 1100, 12, 3, 80, 200, 20),     # with the sinks' far rows apart
    (1, 1100, 1100, 4, 1, 128, 300, 300),    # sinks past those
])
def test_gradients_in_shares(B, Tq, Tk, H, Hkv, D, window, sinks, dt, dev):
    from lockstep_amd.attention import sink_window_attention
    q, k, v, do = inputs(B, Tq, Tk, H, Hkv, D, dt, dev, seed=Tq)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = sink_window_attention(*x, window=window, sinks=sinks)
    grads = torch.autograd.grad(o, x, do, retain_graph=True)
    for b in range(B):
        ref = formula(*(t[b].detach() for t in x), window, sinks, 1.0 / math.sqrt(D), do[b])
        close("o", o[b].detach(), ref["o"], ref["o_mag"], U[dt], 1)
        for n, g in zip(("dq", "dk", "dv"), grads):
            close(n, g[b], ref[n], ref[n + "_mag"], U[dt], 1)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(o, x, do)))


@pytest.mark.parametrize("lens", [[1400], [3, 900, 0, 500], [200] * 9])
def test_packed_gradients_in_shares(lens, dev):
    from lockstep_amd.attention import sink_window_attention
    N, H, Hkv, D = sum(lens) + 5, 8, 1, 128
    q, k, v, do = (t[0] for t in inputs(1, N, N, H, Hkv, D, torch.bfloat16, dev, seed=len(lens)))
    off = [sum(lens[:b]) for b in range(len(lens) + 1)]
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = sink_window_attention(*x, offsets=torch.tensor(off, dtype=torch.int32, device=dev))
    grads = torch.autograd.grad(o, x, do)
    for lo, hi in zip(off, off[1:]):
        if hi > lo:
            ref = formula(*(t[lo:hi].detach() for t in x), None, 0, 1.0 / math.sqrt(D), do[lo:hi])
            close("o", o[lo:hi].detach(), ref["o"], ref["o_mag"], U[torch.bfloat16], 1)
            for n, g in zip(("dq", "dk", "dv"), grads):
                close(n, g[lo:hi], ref[n], ref[n + "_mag"], U[torch.bfloat16], 1)
    assert all((g[off[-1]:] == 0).all() for g in grads)

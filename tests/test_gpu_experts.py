"""experts.expert_gated and expert_combine against their formulas in 64 bits.

Bounds.  The matrix instruction adds eight products at a time and keeps 13
bits below the largest exponent among them: the seven others lose less than
7 * 2^-13 of the largest, so a sum less than that of its magnitudes; over the
eights the sums are fp32.  Where the terms of eight span less than that they
are exact.  The gate has a slope of at most 1.1.  E4M3 rounds by 2^-4 of a
normal value, by half of 2^-9 of the scale below."""

import pytest
import torch

pytestmark = pytest.mark.gpu

IN_BLOCK = 7 * 2.0 ** -13


def _values4(codes, scale):
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device, dtype=torch.float64)
    v = torch.cat([v, -v])
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return v[n] * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def _values8(codes, scale):
    return codes.double() * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def _rows(dev, shape, seed):
    """MXFP8 rows, by the rule, from normal values with channels of different size."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(shape, generator=g, device=dev) * torch.exp(torch.randn(shape[-1], generator=g, device=dev))
    b = x.double().unflatten(-1, (-1, 32))
    e = torch.ceil(torch.log2(b.abs().amax(-1) / 448))
    return (b / torch.exp2(e)[..., None]).flatten(-2).float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _weights(dev, E, N, K, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randint(0, 256, (E, N, K // 2), generator=g, device=dev, dtype=torch.uint8)
    return w, torch.randint(117, 121, (E, N, K // 32), generator=g, device=dev, dtype=torch.uint8)


def _ids(dev, T, k, E, seed, none=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    like = torch.randn((T, E), generator=g, device=dev) + torch.randn(E, generator=g, device=dev)
    ids = like.topk(k, 1).indices.to(torch.int32)
    return torch.where(torch.rand((T, k), generator=g, device=dev) < none, -1, ids).contiguous()


def _products(x, ids, w, ws, slots):
    """[T, k, N] products in 64 bits and the magnitudes added for them."""
    out = torch.zeros((*ids.shape, w.shape[1]), device=x.device, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for e in range(w.shape[0]):
        i, j = torch.nonzero(ids == e, as_tuple=True)
        if i.numel():
            v, rows = _values4(w[e], ws[e]), x[i, j] if slots else x[i]
            out[i, j] = rows @ v.t()
            mag[i, j] = rows.abs() @ v.abs().t()
    return out, mag


# tokens, slots, experts, K, F: one token, few rows for an expert, more than a
# tile's of them, one expert with all, odd numbers, pairs without an expert
GATED = [(1, 1, 1, 128, 32, 0), (1, 4, 32, 256, 64, 0), (5, 2, 3, 384, 96, 0.2), (16, 1, 1, 128, 64, 0), (17, 1, 1, 1408, 32, 0),
         (64, 8, 128, 256, 64, 0.1), (333, 3, 5, 640, 96, 0.1), (130, 2, 2, 128, 160, 0), (600, 4, 4, 512, 128, 0.02),
         (700, 1, 2, 896, 288, 0), (9, 3, 8, 1024, 32, 1.0)]


@pytest.mark.parametrize("T,k,E,K,F,none", GATED)
def test_gated(dev, T, k, E, K, F, none):
    from lockstep_amd import experts
    x, xs = _rows(dev, (T, K), T + K)
    w, ws = _weights(dev, E, 2 * F, K, F)
    ids = _ids(dev, T, k, E, T, none)
    h, hs = experts.expert_gated(x, xs, w, ws, experts.dispatch(ids, E))
    assert h.shape == (T, k, F) and hs.shape == (T, k, F // 32) and h.dtype == torch.float8_e4m3fn
    out, mag = _products(_values8(x, xs), ids, w, ws, False)
    gate, up = out.chunk(2, -1)
    dg, du = (mag * IN_BLOCK).chunk(2, -1)
    want = gate * torch.sigmoid(gate) * up
    err = 1.1 * dg * (up.abs() + du) + (gate * torch.sigmoid(gate)).abs() * du + want.abs() * 2.0 ** -18
    s = torch.exp2(hs.double() - 127)[..., None]
    got = (h.double().unflatten(-1, (-1, 32)) * s).flatten(-2)
    allowed = err * (1 + 2.0 ** -4) + want.abs() * 2.0 ** -4 + (s * 2.0 ** -10).expand(*s.shape[:-1], 32).flatten(-2)
    assert ((got - want).abs() <= allowed).all()
    # the scale is the least that holds the block: its largest code is past 448 / 2 rounded
    top = h.float().unflatten(-1, (-1, 32)).abs().amax(-1)
    there = (ids >= 0)[..., None].expand_as(hs)
    assert (top[there] >= 224).all()
    assert (hs[~there] == 127).all() and (top[~there] == 0).all()


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,k,E,K,N,none", [(1, 1, 1, 128, 1, 0), (1, 4, 32, 256, 64, 0), (5, 2, 3, 384, 100, 0.2), (16, 2, 4, 128, 33, 0),
                                            (17, 4, 4, 1408, 70, 0), (64, 8, 128, 256, 64, 0.1), (333, 3, 5, 640, 130, 0.1),
                                            (600, 4, 4, 512, 257, 0.02), (700, 1, 2, 896, 300, 0), (9, 3, 8, 1024, 32, 1.0), (64, 4, 60, 512, 100, 0.1),
                                            (200, 4, 30, 1152, 513, 0), (300, 2, 9, 768, 770, 0), (2100, 1, 7, 640, 91, 0.3), (40, 3, 1000, 512, 40, 0)])
def test_combine(dev, T, k, E, K, N, none, out_dtype):
    from lockstep_amd import experts
    h, hs = _rows(dev, (T, k, K), T + K)
    w, ws = _weights(dev, E, N, K, N)
    ids = _ids(dev, T, k, E, T, none)
    rw = torch.randn((T, k), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    d = experts.dispatch(ids, E)
    y = experts.expert_combine(h, hs, w, ws, d, rw, out_dtype=out_dtype)
    assert y.shape == (T, N) and y.dtype == out_dtype
    out, mag = _products(_values8(h, hs), ids, w, ws, True)
    c = rw.double()[..., None]
    want, mag = (out * c).sum(1), (mag * c.abs()).sum(1)
    u = torch.finfo(out_dtype).eps / 2
    assert ((y.double() - want).abs() <= want.abs() * u + mag * IN_BLOCK).all()
    assert torch.equal(y, experts.expert_combine(h, hs, w, ws, d, rw, out_dtype=out_dtype))


@pytest.mark.parametrize("T,k,E,K,N", [(3, 2, 4, 256, 96), (40, 2, 3, 512, 130), (500, 2, 3, 384, 256), (1200, 1, 2, 256, 512)])
def test_exact_products(dev, T, k, E, K, N):
    """Codes and scales whose products and sums fp32 holds: equal, bit for bit."""
    from lockstep_amd import experts
    g = torch.Generator(device=dev).manual_seed(K)
    h = torch.randint(-7, 8, (T, k, K), generator=g, device=dev).float().to(torch.float8_e4m3fn)
    hs = torch.randint(125, 129, (T, k, K // 32), generator=g, device=dev, dtype=torch.uint8)
    w, _ = _weights(dev, E, N, K, N)
    ws = torch.randint(126, 129, (E, N, K // 32), generator=g, device=dev, dtype=torch.uint8)
    ids = _ids(dev, T, k, E, T)
    rw = torch.exp2(torch.randint(-1, 2, (T, k), generator=g, device=dev).float())
    y = experts.expert_combine(h, hs, w, ws, experts.dispatch(ids, E), rw, out_dtype=torch.float32)
    want = (_products(_values8(h, hs), ids, w, ws, True)[0] * rw.double()[..., None]).sum(1)
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("T,k,E,K,N", [(3, 2, 4, 256, 96), (40, 2, 16, 1024, 130), (64, 4, 128, 4096, 256), (100, 2, 60, 896, 512)])
def test_few_rows_lose_nothing_in_the_instruction(dev, T, k, E, K, N):
    """Up to 4 rows for an expert, or few workgroups: codes over all of E4M3's range, sums within fp32's
    rounding of K / 8 additions (2^-24 each of the magnitudes, at random: 2^-20)."""
    from lockstep_amd import experts
    g = torch.Generator(device=dev).manual_seed(K)
    codes = torch.randint(0, 256, (T, k, K), generator=g, device=dev, dtype=torch.uint8)
    codes = torch.where((codes & 127) == 127, codes & 128, codes)     # no NaN
    h, hs = codes.view(torch.float8_e4m3fn), torch.randint(120, 130, (T, k, K // 32), generator=g, device=dev, dtype=torch.uint8)
    w, ws = _weights(dev, E, N, K, N)
    ids = torch.arange(T * k, device=dev, dtype=torch.int32).view(T, k) % E
    rw = torch.rand((T, k), generator=g, device=dev)
    y = experts.expert_combine(h, hs, w, ws, experts.dispatch(ids, E), rw, out_dtype=torch.float32)
    out, mag = _products(_values8(h, hs), ids, w, ws, True)
    c = rw.double()[..., None]
    assert ((y.double() - (out * c).sum(1)).abs() <= (mag * c).sum(1) * 2.0 ** -20).all()


def test_nan_scales_and_rows_of_others(dev):
    """A NaN scale or code in one pair's row reaches that pair alone, one in an
    expert's weights that expert's pairs alone."""
    from lockstep_amd import experts
    T, k, E, K, F = 40, 2, 4, 256, 64
    x, xs = _rows(dev, (T, K), 1)
    w, ws = _weights(dev, E, 2 * F, K, 2)
    ids = torch.tensor([[0, 1], [1, 2]] * (T // 2), dtype=torch.int32, device=dev)   # nobody takes expert 3
    d = experts.dispatch(ids, E)
    clean, cs = experts.expert_gated(x, xs, w, ws, d)
    xs2, ws2 = xs.clone(), ws.clone()
    xs2[7, 3] = 255
    ws2[3] = 255
    ws2[2, 5, 1] = 255
    h, hs = experts.expert_gated(x, xs2, w, ws2, d)
    odd = (torch.arange(T, device=dev) == 7)[:, None] | (ids == 2)
    assert torch.equal(h.view(torch.uint8)[~odd], clean.view(torch.uint8)[~odd]) and torch.equal(hs[~odd], cs[~odd])
    assert (hs[7] == 255).all() and (hs[ids == 2][:, 0] == 255).all() and (hs[ids == 2][:, 1] != 255).any()
    z, zs = _rows(dev, (T, k, K), 3)
    w2, w2s = _weights(dev, E, 96, K, 4)
    rw = torch.ones((T, k), device=dev)
    none = ids.clone()
    none[4] = -1
    d = experts.dispatch(none, E)
    zs2 = zs.clone()
    zs2[4] = 255                                          # a row of no expert: not looked at
    rw2 = rw.clone()
    rw2[4] = float("nan")
    y = experts.expert_combine(z, zs, w2, w2s, d, rw)
    y2 = experts.expert_combine(z, zs2, w2, w2s, d, rw2)
    assert torch.equal(y, y2) and (y[4] == 0).all()


def test_a_wrong_dispatch_stays_within_the_tensors(dev):
    """Orders and offsets that no dispatch makes: their pairs may be wrong, the
    call neither fails nor touches anything else."""
    from lockstep_amd import experts
    T, k, E, K, F = 50, 2, 4, 128, 64
    x, xs = _rows(dev, (T, K), 1)
    w, ws = _weights(dev, E, 2 * F, K, 2)
    z, zs = _rows(dev, (T, k, F * 2), 3)
    w2, w2s = _weights(dev, E, 64, F * 2, 4)
    ids = _ids(dev, T, k, E, 5)
    good = experts.dispatch(ids, E)
    rw = torch.ones((T, k), device=dev)
    for order, offsets in ((good.order + 10 ** 6, good.offsets), (-good.order - 1, good.offsets), (good.order, good.offsets.flip(0)),
                           (good.order, good.offsets * 1000 - 7), (good.order, torch.full_like(good.offsets, 100))):
        d = experts.Dispatch(ids, order.contiguous(), offsets.contiguous())
        experts.expert_gated(x, xs, w, ws, d)
        experts.expert_combine(z, zs, w2, w2s, d, rw)
    torch.cuda.synchronize()
    h = experts.expert_gated(x, xs, w, ws, good)[0]
    assert torch.isfinite(h.float()).all()


def test_shapes_strides_and_empty_calls(dev):
    from lockstep_amd import experts
    T, k, E, K, F = 24, 2, 4, 256, 128
    x, xs = _rows(dev, (T, K), 1)
    w, ws = _weights(dev, E, 2 * F, K, 2)
    w2, w2s = _weights(dev, E, 64, F, 3)
    ids = _ids(dev, T, k, E, 5)
    rw = torch.rand((T, k), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    d = experts.dispatch(ids, E)
    h, hs = experts.expert_gated(x, xs, w, ws, d)
    y = experts.expert_combine(h, hs, w2, w2s, d, rw)
    # leading axes, bytes for codes, strides
    d3 = experts.dispatch(ids.view(4, 6, k), E)
    h3, hs3 = experts.expert_gated(x.view(torch.uint8).view(4, 6, K), xs.view(4, 6, -1), w, ws, d3)
    assert h3.shape == (4, 6, k, F) and torch.equal(h3.view(torch.uint8).flatten(0, 1), h.view(torch.uint8))
    y3 = experts.expert_combine(h3, hs3, w2, w2s, d3, rw.view(4, 6, k))
    assert y3.shape == (4, 6, 64) and torch.equal(y3.flatten(0, 1), y)
    wide = torch.zeros((T, K + 5), dtype=torch.uint8, device=dev)
    wide[:, 3:K + 3] = x.view(torch.uint8)
    sw = ws.transpose(1, 2).contiguous().transpose(1, 2)
    h4, hs4 = experts.expert_gated(wide[:, 3:K + 3].view(torch.float8_e4m3fn), xs, w, sw, d)
    assert torch.equal(h4.view(torch.uint8), h.view(torch.uint8)) and torch.equal(hs4, hs)
    # no tokens
    d0 = experts.dispatch(ids[:0], E)
    h0, hs0 = experts.expert_gated(x[:0], xs[:0], w, ws, d0)
    assert h0.shape == (0, k, F) and hs0.shape == (0, k, F // 32) and d0.offsets.tolist() == [0] * (E + 1)
    assert experts.expert_combine(h0, hs0, w2, w2s, d0, rw[:0]).shape == (0, 64)
    # one token without axes
    d1 = experts.dispatch(ids[3], E)
    h1, hs1 = experts.expert_gated(x[3], xs[3], w, ws, d1)
    assert torch.equal(h1.view(torch.uint8), h[3].view(torch.uint8))
    assert experts.expert_combine(h1, hs1, w2, w2s, d1, rw[3]).shape == (64,)


@pytest.mark.parametrize("T", [3, 300])
def test_a_layer_as_it_is_used(dev, T):
    """Norm, router, dispatch and both products in a run, eagerly, on another
    stream and replayed, against the formulas on the values each step made."""
    from lockstep_amd import experts, fp4
    from lockstep_amd.norm import add_rms_norm
    D, F, E, k = 256, 128, 16, 4
    g = torch.Generator(device=dev).manual_seed(T)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    x, r, nw = rnd(T, D).bfloat16(), rnd(T, D).bfloat16(), (1 + 0.1 * rnd(D)).bfloat16()
    router, bias = 0.1 * rnd(E, D).bfloat16(), 0.05 * rnd(E)
    w13, s13 = fp4.quantize_pack_mxfp4((0.06 * rnd(E, 2 * F, D)).bfloat16())
    w2, s2 = fp4.quantize_pack_mxfp4((0.1 * rnd(E, D, F)).bfloat16())

    def layer():
        y, h, x8, xs = add_rms_norm(x, nw, r, mxfp8=True)
        weights, ids = experts.route(y @ router.t(), k, scoring="sigmoid", bias=bias, groups=4, top_groups=2, scale=2.5)
        d = experts.dispatch(ids, E)
        a, s = experts.expert_gated(x8, xs, w13, s13, d)
        return x8, xs, ids, weights, a, s, experts.expert_combine(a, s, w2, s2, d, weights), h

    x8, xs, ids, weights, a, s, out, h = got = layer()
    up, mag = _products(_values8(x8, xs), ids, w13, s13, False)
    gate, lin = up.chunk(2, -1)
    want = gate * torch.sigmoid(gate) * lin
    have = _values8(a, s)
    dg, du = (mag * IN_BLOCK).chunk(2, -1)
    err = 1.1 * dg * (lin.abs() + du) + (gate * torch.sigmoid(gate)).abs() * du
    step = torch.exp2(s.double() - 127).repeat_interleave(32, -1) * 2.0 ** -10
    assert ((have - want).abs() <= 1.1 * err + want.abs() * (2.0 ** -4 + 2.0 ** -18) + step).all()
    p, mag = _products(have, ids, w2, s2, True)
    c = weights.double()[..., None]
    assert ((out.double() - (p * c).sum(1)).abs() <= (p * c).sum(1).abs() * 2.0 ** -8 + (mag * c).sum(1) * IN_BLOCK).all()
    same = lambda u, v: all(torch.equal(i.view(torch.uint8), j.view(torch.uint8)) for i, j in zip(u, v))  # noqa: E731
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = layer()
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            held = layer()
    assert same(other, got)
    for i in range(3):
        x.copy_(rnd(T, D))
        graph.replay()
        torch.cuda.synchronize()
        assert same(held, layer())


@pytest.mark.parametrize("T,k,E,K,N", [(30, 1, 1, 512, 64), (60, 2, 1, 640, 130), (100, 1, 2, 1024, 192), (384, 1, 4, 512, 33), (97, 1, 1, 512, 257)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_many_rows_of_few_experts_in_few_workgroups(dev, T, k, E, K, N, out_dtype):
    """Where the rows of an expert are many, but its rows of W few."""
    from lockstep_amd import experts
    h, hs = _rows(dev, (T, k, K), T + K)
    w, ws = _weights(dev, E, N, K, N)
    ids = _ids(dev, T, k, E, T) if k <= E else torch.zeros((T, k), dtype=torch.int32, device=dev)
    rw = torch.randn((T, k), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    y = experts.expert_combine(h, hs, w, ws, experts.dispatch(ids, E), rw, out_dtype=out_dtype)
    out, mag = _products(_values8(h, hs), ids, w, ws, True)
    c = rw.double()[..., None]
    want, mag = (out * c).sum(1), (mag * c.abs()).sum(1)
    assert ((y.double() - want).abs() <= want.abs() * torch.finfo(out_dtype).eps / 2 + mag * (IN_BLOCK + 2.0 ** -11)).all()


def test_large_blocks_large_weights_and_zeros(dev):
    """bf16 sums of many rows at the ends of fp32: a row of W that is zero gives 0
    beside one that gives 2^120, whatever the weight; an infinite product stays one."""
    from lockstep_amd import experts
    T, E, K, N = 200, 1, 512, 320
    h = torch.full((T, 1, K), 2.0, device=dev).to(torch.float8_e4m3fn)
    hs = torch.full((T, 1, K // 32), 127, dtype=torch.uint8, device=dev)
    hs[50:] = 127 + 100
    w = torch.full((E, N, K // 2), 0x22, dtype=torch.uint8, device=dev)      # ones
    w[:, ::2] = 0
    ws = torch.full((E, N, K // 32), 127 + 10, dtype=torch.uint8, device=dev)
    ids = torch.zeros((T, 1), dtype=torch.int32, device=dev)
    rw = torch.full((T, 1), 2.0 ** 5, device=dev)
    rw[100:] = 2.0 ** -100
    rw[150:] = 2.0 ** 17        # with 2^120: infinite, and 2^17 beside the block's scale
    y = experts.expert_combine(h, hs, w, ws, experts.dispatch(ids, E), rw)
    want = torch.zeros((T, N), dtype=torch.float64, device=dev)
    want[:50, 1::2], want[50:100, 1::2], want[100:150, 1::2] = 2.0 ** 25, 2.0 ** 125, 2.0 ** 20
    want[150:, 1::2] = float("inf")
    assert torch.equal(y.double(), want)

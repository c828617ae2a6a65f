"""The MXFP4 cache: append, attention over it, accumulated weights, eviction.

Tolerances.  The values held are exact (E2M1 times a power of two), so the
formula in 64 bits starts from them.  o: each probability is rounded once to
the rows' type and the result once, so
|err| <= 4 u sum_j p_j |v_j| with u = 2^-8 (bf16) or 2^-11 (fp16) has room
for the fp32 sums.  weights stay in fp32: a score's error is at most
2^-20 (1 + scale sum |q_d k_d|) with room (chains of at most 128 terms in
fp32), which is the relative error of its probability and of the row's sum."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def scattered(counts, dev, seed, spare=0, first=0):
    """A block table over a shuffled pool, -7 past each sequence's pages."""
    n = sum(counts)
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(n + spare, generator=g)[:n].to(torch.int32) + first
    table = torch.full((len(counts), max(counts + [1])), -7, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return table.to(dev), first + n + spare


def filled(lens, Hkv, D, page, dt, dev, seed=0):
    """A cache of the given lengths, and the values it holds [len, Hkv, D]."""
    from lockstep_amd import kv_cache as kc
    g = torch.Generator(device=dev).manual_seed(seed)
    table, n = scattered([-(-x // page) for x in lens], dev, seed, spare=3)
    pages = kc.new_pages(n, Hkv, D, page, device=dev)
    for t in pages:   # what was in the pool before must not matter
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=dev, dtype=torch.uint8))
    N = sum(lens)
    k = (torch.randn((N, Hkv, D), generator=g, device=dev) * torch.exp(torch.randn((Hkv, D), generator=g, device=dev))).to(dt)
    v = torch.randn((N, Hkv, D), generator=g, device=dev).to(dt)
    off = torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    kv = kc.append(pages, k, v, table, lengths, offsets=off, values=True)
    split = [[x[sum(lens[:b]):sum(lens[:b + 1])] for b in range(len(lens))] for x in kv]
    return pages, table, lengths, split, (k, v)


def held(pages, table, b, n, page, dev):
    """Codes and scales of sequence b, in token order."""
    j = torch.arange(n, device=dev)
    pg = table[b, j // page].long()
    return [t[pg, :, j % page] for t in pages]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,Hkv,D,page", [([1], 1, 64, 16), ([16, 0, 33], 3, 128, 16), ([100, 257, 5], 2, 64, 64),
                                             ([70] * 70, 1, 64, 32), ([2050], 8, 128, 1024)])
def test_append_holds_the_quantizers_bytes(lens, Hkv, D, page, dt, dev):
    from lockstep_amd import fp4
    pages, table, lengths, (kv, vv), (k, v) = filled(lens, Hkv, D, page, dt, dev, seed=len(lens))
    at = 0
    for b, n in enumerate(lens):
        got = held(pages, table, b, n, page, dev)
        for x, c, s, val in ((k, got[0], got[1], kv), (v, got[2], got[3], vv)):
            x = x[at:at + n]
            if n == 0:
                continue
            pk, e8 = fp4.quantize_pack_mxfp4(x.contiguous())
            assert torch.equal(c, pk) and torch.equal(s, e8)
            codes, sc = fp4.quantize_mxfp4(x.contiguous())
            assert torch.equal(val[b].float(), fp4.dequantize_mxfp4(codes, sc))
        at += n


def test_append_edges(dev):
    """Zero, Inf and NaN blocks, padding in front, positions past the table,
    ids outside the pool, offset-free form, strided inputs."""
    from lockstep_amd import fp4
    from lockstep_amd import kv_cache as kc
    pages = kc.new_pages(4, 2, 64, 16, device=dev)
    x = torch.randn((3, 20, 2, 64), device=dev).half()
    x[0, 3, 0, :32] = 0
    x[0, 4, 1, 5] = float("inf")
    x[0, 5, 1, 40] = float("nan")
    x[1, :, :, 0] = -0.0
    y = torch.randn((3, 20, 2, 2, 64), device=dev).half()[:, :, :, 1]       # strided
    table = torch.tensor([[2, 0], [9, 3], [-1, 1]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([20, 40, 7], dtype=torch.int32, device=dev)      # 1: past the table; 2: 13 in front
    kv, vv = kc.append(pages, x, y, table, lengths, values=True)
    assert kv.shape == x.shape and kv.dtype == torch.bfloat16
    want = fp4.quantize_pack_mxfp4(x.contiguous()), fp4.quantize_pack_mxfp4(y.contiguous())
    written = torch.zeros((4, 16), dtype=torch.bool, device=dev)
    for b, n in enumerate(lengths.tolist()):
        for i in range(20):
            j = n - 20 + i
            if not 0 <= j < 32 or not 0 <= table[b, j // 16].item() < 4:
                continue
            p = table[b, j // 16].item()
            written[p, j % 16] = True
            for o, w in ((0, want[0]), (2, want[1])):
                assert torch.equal(pages[o][p, :, j % 16], w[0][b, i]), (b, i)
                assert torch.equal(pages[o + 1][p, :, j % 16], w[1][b, i])
    for t in pages:
        assert (t.permute(0, 2, 1, 3)[~written] == 0).all()
    # offset-free equals packed
    p2 = kc.new_pages(4, 2, 64, 16, device=dev)
    off = torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=dev)
    kc.append(p2, x.reshape(60, 2, 64), y.reshape(60, 2, 64), table, lengths, offsets=off)
    assert all(torch.equal(a, b) for a, b in zip(pages, p2))


def formula(q, k, v, window, sinks, scale):
    """One sequence: q [T, H, D], k, v [n, Hkv, D] -> o, its magnitudes, the
    weights [Hkv, n] and the bound on their error."""
    T, H, _ = q.shape
    n, Hkv, _ = k.shape
    G = H // Hkv
    q, k, v = q.double().transpose(0, 1), k.double().transpose(0, 1), v.double().transpose(0, 1)
    kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    p = torch.arange(T, device=q.device)[:, None] + n - T
    j = torch.arange(n, device=q.device)[None]
    see = j <= p
    if window is not None:
        see = see & ((j > p - window) | (j < sinks))
    s = torch.where(see, scale * (q @ kk.transpose(1, 2)), -math.inf)
    m = s.amax(-1, keepdim=True) if n else s.new_full((H, T, 1), -math.inf)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m)) * see
    tot = e.sum(-1, keepdim=True)
    w = e / torch.where(tot == 0, 1.0, tot)
    mag = 1 + scale * (q.abs() @ kk.abs().transpose(1, 2))
    err = 2.0 ** -20 * w * (mag + (w * mag).sum(-1, keepdim=True))
    fold = lambda x: x.unflatten(0, (Hkv, G)).sum((1, 2))  # noqa: E731
    return (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1), fold(w), fold(err)


CASES = [
    # lens, T, H, Hkv, D, page, window, sinks
    ([1], 1, 1, 1, 64, 16, None, 0),
    ([1000], 1, 32, 8, 128, 16, None, 0),
    ([31, 0, 32, 33, 500], 1, 4, 2, 64, 16, None, 0),
    ([5, 300], 4, 6, 1, 128, 32, None, 0),           # 24 rows
    ([3, 1, 129], 5, 10, 1, 64, 64, None, 0),        # rows before the first token
    ([700, 64], 1, 8, 2, 128, 64, 50, 0),
    ([700, 64, 10], 2, 20, 1, 128, 64, 33, 40),      # 40 rows, sinks over two tiles
    ([3000, 2777], 1, 5, 1, 128, 256, None, 0),      # few heads, split
    ([2500], 3, 16, 1, 64, 16, 2000, 4),
    ([200, 90, 30], 65, 4, 2, 128, 32, None, 0),     # tiles of 128 rows
    ([650, 129], 129, 6, 2, 64, 16, 100, 5),
    ([300], 300, 3, 3, 128, 1024, 1, 2),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_attend(case, dt, dev):
    from lockstep_amd import kv_cache as kc
    lens, T, H, Hkv, D, page, window, sinks = case
    pages, table, lengths, (kv, vv), _ = filled(lens, Hkv, D, page, dt, dev, seed=T + D)
    g = torch.Generator(device=dev).manual_seed(11)
    q = torch.randn((len(lens), T, H, D), generator=g, device=dev).to(dt)
    w0 = torch.rand((len(lens), Hkv, table.shape[1] * page + 3), generator=g, device=dev)
    w = w0.clone()
    o = kc.attend(q, pages, table, lengths, window=window, sinks=sinks, weights=w)
    assert torch.equal(o, kc.attend(q, pages, table, lengths, window=window, sinks=sinks))
    for b, n in enumerate(lens):
        ro, mag, rw, err = formula(q[b], kv[b], vv[b], window, sinks, 1.0 / math.sqrt(D))
        bad = (o[b].double() - ro).abs() - (4 * U[dt] * mag + 1e-7)
        assert torch.isfinite(o[b]).all() and bad.max().item() <= 0, (b, bad.max().item())
        new = w0[b].double()
        new[:, :n] += rw
        tol = 2.0 ** -22 * new.abs()
        tol[:, :n] += err
        bad = (w[b].double() - new).abs() - tol
        assert bad.max().item() <= 0, (b, bad.max().item())


def test_attend_long_split_and_far_pages(dev):
    """A cache whose pool passes 2^31 bytes: offsets beyond 32 bits, in both
    forms (few rows, many rows)."""
    from lockstep_amd import kv_cache as kc
    Hkv, D, page = 8, 128, 1024
    n = 4200                                          # 4200 x 8 x 1024 x 64 B = 2.2 GB of codes
    pages = kc.new_pages(n, Hkv, D, page, device=dev)
    table = torch.tensor([[n - 1, 1, n - 2]], dtype=torch.int32, device=dev)
    lens = torch.tensor([2600], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    k, v = (torch.randn((1, 2600, Hkv, D), generator=g, device=dev).bfloat16() for _ in range(2))
    kv, vv = kc.append(pages, k, v, table, lens, values=True)
    for T in (1, 70):
        q = torch.randn((1, T, 16, D), generator=g, device=dev).bfloat16()
        o = kc.attend(q, pages, table, lens)
        ro, mag, _, _ = formula(q[0], kv[0], vv[0], None, 0, 1.0 / math.sqrt(D))
        assert ((o[0].double() - ro).abs() <= 4 * 2.0 ** -8 * mag + 1e-7).all()
    del pages
    torch.cuda.empty_cache()


def test_hidden_pages_and_nan_tokens(dev):
    """An id outside the pool hides its tokens; NaN in tokens that a row's
    window hides does not reach it in another 64-token tile; scales of NaN
    past a sequence's end do nothing."""
    from lockstep_amd import kv_cache as kc
    pages, table, lengths, (kv, vv), _ = filled([200], 2, 64, 16, torch.bfloat16, dev, seed=4)
    g = torch.Generator(device=dev).manual_seed(1)
    for T in (1, 80):
        q = torch.randn((1, T, 4, 64), generator=g, device=dev).bfloat16()
        t2 = table.clone()
        t2[0, 3] = 10 ** 6
        t2[0, 5] = -1
        w = torch.zeros((1, 2, t2.shape[1] * 16), device=dev)
        o = kc.attend(q, pages, t2, lengths, weights=w)
        hide = torch.zeros(200, dtype=torch.bool, device=dev)
        hide[48:64] = hide[80:96] = True
        qd = q[0].double().transpose(0, 1)
        kk = kv[0].double().transpose(0, 1).repeat_interleave(2, 0)
        s = (qd @ kk.transpose(1, 2)) / 8.0
        pos = torch.arange(T, device=dev)[:, None] + 200 - T
        s = s.masked_fill(hide | (torch.arange(200, device=dev)[None] > pos), -math.inf)
        p = torch.softmax(s, -1)
        ref = (p @ vv[0].double().transpose(0, 1).repeat_interleave(2, 0)).transpose(0, 1)
        assert ((o[0].double() - ref).abs() <= 0.02).all()
        assert (w[0][:, :200][:, hide] == 0).all()
        assert abs(w.sum().item() - 4 * T) <= 1e-3 * 4 * T
    # NaN tokens far outside the window
    pages[1][table[0, 0].long()] = 255
    pages[3][table[0, 0].long()] = 255
    for T in (1, 80):
        q = torch.randn((1, T, 4, 64), generator=g, device=dev).bfloat16()
        assert torch.isfinite(kc.attend(q, pages, table, lengths, window=30)).all()
        assert torch.isnan(kc.attend(q, pages, table, lengths)).any()


def reference_evict(w, n, keep, sinks, recent):
    if n <= keep:
        return list(range(n))
    c0, c1 = min(sinks, n), max(min(sinks, n), n - recent)
    key = lambda j: (0 if math.isnan(w[j]) else 1, -w[j] if not math.isnan(w[j]) else 0, j)  # noqa: E731
    best = sorted(range(c0, c1), key=key)[:keep - (n - (c1 - c0))]
    return sorted(list(range(c0)) + best + list(range(c1, n)))


@pytest.mark.parametrize("lens,Hkv,D,page,keep,sinks,recent,kind", [
    ([1], 1, 64, 16, 1, 0, 0, "rand"),
    ([40, 0, 17], 2, 64, 16, 17, 1, 4, "rand"),
    ([300, 299, 64], 3, 128, 32, 64, 4, 30, "ties"),
    ([2000, 1025], 2, 128, 64, 1024, 0, 0, "rand"),
    ([1500], 1, 64, 256, 700, 100, 600, "rand"),      # the protected alone
    ([5000], 2, 64, 64, 1, 0, 0, "odd"),
    ([3000, 2049], 1, 128, 16, 1100, 3, 64, "odd"),
    ([700], 2, 64, 16, 300, 0, 300, "ties"),          # no candidate stays
])
def test_evict(lens, Hkv, D, page, keep, sinks, recent, kind, dev):
    from lockstep_amd import kv_cache as kc
    pages, table, lengths, _, _ = filled(lens, Hkv, D, page, torch.bfloat16, dev, seed=keep)
    B, cap = len(lens), table.shape[1] * page
    g = torch.Generator(device=dev).manual_seed(keep)
    w = torch.exp(3 * torch.randn((B, Hkv, cap + 5), generator=g, device=dev))
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=g, device=dev).float()
    if kind == "odd":   # every sort of value
        pick = torch.tensor([0.0, -0.0, 1e-40, -1.0, 2.5, float("inf"), -float("inf"), float("nan"), 3e38, -3e38], device=dev)
        w = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.7,
                        pick[torch.randint(0, 10, w.shape, generator=g, device=dev)], w)
    spare = -(-min(keep, cap) // page)
    n0 = pages[0].shape[0]
    grown = kc.Pages(*(torch.cat([t, torch.zeros((B * spare, *t.shape[1:]), dtype=t.dtype, device=dev)]) for t in pages))
    out_table = (torch.randperm(B * spare).to(torch.int32) + n0).reshape(B, spare).to(dev)
    before = [t.clone() for t in grown]
    index, kept, new = kc.evict(grown, table, lengths, w, keep, out_table, sinks=sinks, recent=recent)
    assert new.tolist() == [min(n, keep) for n in lens]
    wl = w.cpu().tolist()
    for b, n in enumerate(lens):
        src = held(before, table, b, n, page, dev)
        for h in range(Hkv):
            want = reference_evict(wl[b][h], n, keep, sinks, recent)
            m = len(want)
            assert index[b, h].tolist() == want + [-1] * (keep - m)
            at = torch.tensor(want, device=dev, dtype=torch.long)
            assert torch.equal(kept[b, h, :m].view(torch.int32), w[b, h, at].view(torch.int32))
            assert (kept[b, h, m:] == 0).all()
            dst = held(grown, out_table, b, m, page, dev)
            for s, d in zip(src, dst):
                assert torch.equal(s[at, h], d[:, h])
    for t, t0 in zip(grown, before):   # the old pages are as they were
        assert torch.equal(t[:n0], t0[:n0])


def test_decode_loop_with_eviction(dev):
    """The operators in turn: fill, decode with weights, evict, decode on."""
    from lockstep_amd import kv_cache as kc
    B, H, Hkv, D, page, keep = 2, 4, 2, 64, 16, 48
    g = torch.Generator(device=dev).manual_seed(7)
    pages = kc.new_pages(40, Hkv, D, page, device=dev)
    table = torch.arange(16, dtype=torch.int32, device=dev).reshape(B, 8)
    other = torch.arange(20, 36, dtype=torch.int32, device=dev).reshape(B, 8)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    w = torch.zeros((B, Hkv, 128), device=dev)
    ks, vs = [[[] for _ in range(Hkv)] for _ in range(B)], [[[] for _ in range(Hkv)] for _ in range(B)]
    for step in range(150):
        r = lambda h: torch.randn((B, 1, h, D), generator=g, device=dev).bfloat16()  # noqa: E731
        q, k, v = r(H), r(Hkv), r(Hkv)
        lengths += 1
        kv, vv = kc.append(pages, k, v, table, lengths, values=True)
        o = kc.attend(q, pages, table, lengths, sinks=2, weights=w)
        for b in range(B):
            for h in range(Hkv):
                ks[b][h].append(kv[b, 0, h])
                vs[b][h].append(vv[b, 0, h])
                ro, mag, _, _ = formula(q[b][:, 2 * h:2 * h + 2], torch.stack(ks[b][h])[:, None],
                                        torch.stack(vs[b][h])[:, None], None, 0, 0.125)
                assert ((o[b][:, 2 * h:2 * h + 2].double() - ro).abs() <= 4 * 2.0 ** -8 * mag + 1e-7).all(), step
        if lengths[0].item() == 100:
            index, kept, lengths = kc.evict(pages, table, lengths, w, keep, other, sinks=2, recent=8)
            table, other = other, table
            w = torch.zeros_like(w)
            w[:, :, :keep] = kept
            for b in range(B):
                for h in range(Hkv):
                    at = index[b, h].tolist()
                    ks[b][h], vs[b][h] = [ks[b][h][j] for j in at], [vs[b][h][j] for j in at]


def test_graph_capture_and_streams(dev):
    """A captured decode step replays on new contents, with eager work between."""
    from lockstep_amd import kv_cache as kc
    pages, table, lengths, _, _ = filled([900, 400], 2, 128, 64, torch.bfloat16, dev, seed=1)
    table = torch.nn.functional.pad(table, (0, 1), value=-1).contiguous()
    q = torch.randn((2, 1, 8, 128), device=dev).bfloat16()
    k, v = (torch.randn((2, 1, 2, 128), device=dev).bfloat16() for _ in range(2))
    w = torch.zeros((2, 2, table.shape[1] * 64), device=dev)
    def step():
        kc.append(pages, k, v, table, lengths)
        return kc.attend(q, pages, table, lengths, weights=w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step().clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(step(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        q.copy_(torch.randn((2, 1, 8, 128), device=dev))
        k.copy_(torch.randn((2, 1, 2, 128), device=dev))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, gw = out.clone(), w.clone()
        w.zero_()
        assert torch.equal(step(), got) and torch.equal(w, gw), i


def test_refused(dev):
    from lockstep_amd import kv_cache as kc
    pages = kc.new_pages(4, 2, 64, 16, device=dev)
    table = torch.zeros((1, 2), dtype=torch.int32, device=dev)
    lengths = torch.tensor([5], dtype=torch.int32, device=dev)
    q = torch.zeros((1, 1, 4, 64), dtype=torch.bfloat16, device=dev)
    k = torch.zeros((1, 1, 2, 64), dtype=torch.bfloat16, device=dev)
    w = torch.zeros((1, 2, 32), device=dev)
    for page in (8, 24, 2048):
        with pytest.raises(AssertionError):
            kc.new_pages(1, 1, 64, page, device=dev)
    with pytest.raises(AssertionError):
        kc.new_pages(1, 1, 96, 16, device=dev)
    with pytest.raises(TypeError):
        kc.attend(q.float(), pages, table, lengths)
    with pytest.raises(AssertionError):
        kc.attend(q[:, :, :3], pages, table, lengths)
    with pytest.raises(AssertionError):
        kc.attend(q, pages, table.long(), lengths)
    with pytest.raises(AssertionError):
        kc.attend(q, pages, table, lengths.long())
    with pytest.raises(AssertionError):
        kc.attend(q, pages, table, lengths, weights=w[:, :, :31].contiguous())
    with pytest.raises(AssertionError):
        kc.attend(q, pages, table, lengths, weights=w.half())
    with pytest.raises(AssertionError):
        kc.attend(q, kc.Pages(pages[0][:, :, :, ::2], *pages[1:]), table, lengths)
    with pytest.raises(ValueError):
        kc.attend(q, pages, table, lengths, window=0)
    with pytest.raises(RuntimeError):
        kc.attend(q.cpu(), pages, table, lengths)
    with pytest.raises(TypeError):
        kc.append(pages, k.float(), k.float(), table, lengths)
    with pytest.raises(AssertionError):
        kc.append(pages, k, k[:, :, :1], table, lengths)
    with pytest.raises(AssertionError):
        kc.append(pages, k[0], k[0], table, lengths)
    with pytest.raises(AssertionError):
        kc.append(pages, k[0], k[0], table, lengths, offsets=torch.zeros(3, dtype=torch.int32, device=dev))
    out = torch.ones((1, 2), dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        kc.evict(pages, table, lengths, w, 0, out)
    with pytest.raises(ValueError):
        kc.evict(pages, table, lengths, w, 4, out, sinks=3, recent=2)
    with pytest.raises(AssertionError):
        kc.evict(pages, table, lengths, w, 20, out[:, :1].contiguous())
    with pytest.raises(AssertionError):
        kc.evict(pages, table, lengths, w[:, :1].contiguous(), 4, out)
    # empty calls
    assert kc.attend(q[:0], pages, table[:0], lengths[:0]).shape == (0, 1, 4, 64)
    assert kc.attend(q[:, :0], pages, table, lengths).shape == (1, 0, 4, 64)
    assert kc.append(pages, k[:, :0], k[:, :0], table, lengths, values=True)[0].shape == (1, 0, 2, 64)
    none = torch.zeros((1, 0), dtype=torch.int32, device=dev)
    assert (kc.attend(q, pages, none, lengths) == 0).all()

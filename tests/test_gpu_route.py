"""experts.route and dispatch against their definitions in 64 bits.

The choice has to be the definition's, index by index.  Weights are fp32 of
scores in at least fp32 precision: 2^-20 of the value covers the score's
rounding, k <= 64 additions and a division.  Gradients: half a step of the
logits' type and 2^-20 of the magnitudes that are added."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _route64(logits, k, bias, scoring, groups, top_groups, renorm, scale):
    x = logits.double()
    s = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    rank = s if bias is None else s + bias.double()
    if groups > 1:
        by = rank.unflatten(-1, (groups, -1))
        two = torch.sort(by, dim=-1, descending=True, stable=True).values[..., :2].sum(-1)
        top = torch.sort(two, dim=-1, descending=True, stable=True).indices[..., :top_groups]
        keep = torch.zeros_like(two, dtype=torch.bool).scatter(-1, top, True)
        rank = by.masked_fill(~keep[..., None], -float("inf")).flatten(-2)
    at = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :k]
    a = s.gather(-1, at)
    return scale * (a / a.sum(-1, keepdim=True) if renorm else a), at


def _logits(dev, T, E, dt, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (1.5 * torch.randn((T, E), generator=g, device=dev) + 0.5 * torch.randn(E, generator=g, device=dev)).to(DT[dt])


SHAPES = [(1, 1, 1, 1, 1), (5, 2, 2, 1, 1), (33, 8, 2, 1, 1), (7, 60, 4, 1, 1), (130, 64, 6, 1, 1), (9, 65, 8, 5, 2),
          (64, 256, 8, 8, 4), (31, 240, 8, 8, 3), (11, 160, 6, 8, 8), (6, 384, 8, 1, 1), (5, 512, 10, 16, 4), (3, 1024, 64, 64, 4),
          (4, 1000, 64, 1, 1), (17, 64, 5, 64, 7)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k,groups,top", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_choice_and_weights(dev, dt, T, E, k, groups, top, scoring, bias):
    from lockstep_amd.experts import route
    logits = _logits(dev, T, E, dt, E + k)
    b = 0.1 * torch.randn(E, generator=torch.Generator(device=dev).manual_seed(1), device=dev) if bias else None
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        w, ids = route(logits, k, bias=b, scoring=scoring, groups=groups, top_groups=top, renormalize=renorm, scale=scale)
        want, at = _route64(logits, k, b, scoring, groups, top, renorm, scale)
        assert ids.dtype == torch.int32 and torch.equal(ids.long(), at)
        assert ((w.double() - want).abs() <= want * 2.0 ** -20).all()


def test_ties_go_to_the_lowest_index(dev):
    from lockstep_amd.experts import route
    logits = torch.zeros((3, 96), device=dev)
    logits[1, 40] = logits[1, 41] = logits[1, 95] = 1.0
    logits[2] = torch.arange(96, device=dev) % 3
    for scoring in ("softmax", "sigmoid"):
        _, ids = route(logits, 4, scoring=scoring)
        assert ids.tolist() == [[0, 1, 2, 3], [40, 41, 95, 0], [2, 5, 8, 11]]
        _, ids = route(logits, 4, scoring=scoring, groups=4, top_groups=2)
        assert ids[0].tolist() == [0, 1, 2, 3] and ids[1].tolist() == [40, 41, 95, 24]
        _, ids = route(logits, 3, scoring=scoring, bias=torch.zeros(96, device=dev))
        assert ids[0].tolist() == [0, 1, 2]


def test_choices_nearer_than_32_bits(dev):
    """Scores that are equal in 32 bits and differ in 64: the definition's order."""
    from lockstep_amd.experts import route
    g = torch.Generator(device=dev).manual_seed(3)
    E = 64
    logits = torch.randn((200, E), generator=g, device=dev)
    logits[:, 1::2] = logits[:, ::2]                     # pairs of one score ..
    step = torch.randint(-2, 3, (200, E // 2), generator=g, device=dev, dtype=torch.int32)
    near = (logits[:, ::2].view(torch.int32) + step).view(torch.float32)
    logits[:, 1::2] = near                               # .. up to two steps of fp32 apart
    bias = torch.randn(E // 2, generator=g, device=dev).repeat_interleave(2)
    for scoring in ("softmax", "sigmoid"):
        for groups, top in ((1, 1), (8, 3)):
            w, ids = route(logits, 8, scoring=scoring, bias=bias, groups=groups, top_groups=top)
            assert torch.equal(ids.long(), _route64(logits, 8, bias, scoring, groups, top, True, 1.0)[1])
            w, ids = route(logits, 8, scoring=scoring, groups=groups, top_groups=top)
            assert torch.equal(ids.long(), _route64(logits, 8, None, scoring, groups, top, True, 1.0)[1])


def test_infinities_nan_and_masked_rows(dev):
    from lockstep_amd.experts import route
    inf, nan = float("inf"), float("nan")
    logits = torch.zeros((6, 8), device=dev)
    logits[0] = -inf                                     # nothing: scores of 0
    logits[1, :6] = -inf                                 # two experts left for three places
    logits[2, 5] = nan
    logits[3, 2] = inf
    logits[4] = torch.finfo(torch.float32).min           # equal, however low
    w, ids = route(logits, 3)
    assert ids[0].tolist() == [0, 1, 2] and w[0].tolist() == [0, 0, 0]
    assert ids[1].tolist() == [6, 7, 0] and w[1].tolist() == [0.5, 0.5, 0]
    assert torch.isnan(w[2]).all() and torch.isnan(w[3]).all()
    assert ids[4].tolist() == [0, 1, 2] and (w[4] - 1 / 3).abs().max() < 1e-6
    w, ids = route(logits, 3, scoring="sigmoid")
    assert ids[0].tolist() == [0, 1, 2] and w[0].tolist() == [0, 0, 0]
    assert ids[2].tolist() == [5, 0, 1] and ids[3].tolist() == [2, 0, 1] and w[3].tolist() == [0.5, 0.25, 0.25]
    assert ((ids >= 0) & (ids < 8)).all()
    mask = torch.tensor([False, True, False, True, True, False], device=dev)
    lg = logits.clone().requires_grad_(True)
    for scoring in ("softmax", "sigmoid"):
        w, ids = route(lg, 3, mask=mask, scoring=scoring)
        assert (ids[~mask] == -1).all() and (w[~mask] == 0).all() and (ids[mask] >= 0).all()
        d, = torch.autograd.grad(w, lg, torch.ones_like(w))
        assert (d[~mask] == 0).all() and d[4].abs().max() < 1e-6


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 8, 2), (33, 60, 4), (9, 130, 8), (4, 300, 3), (2, 1024, 64), (1025, 64, 6)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient(dev, dt, T, E, k, scoring, renorm):
    from lockstep_amd.experts import route
    logits = _logits(dev, T, E, dt, E).requires_grad_(True)
    w, ids = route(logits, k, scoring=scoring, renormalize=renorm, scale=1.5)
    up = torch.randn((T, k), generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    d, = torch.autograd.grad(w, logits, up)
    x = logits.detach().double().requires_grad_(True)
    s = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    a = s.gather(-1, ids.long())
    want, = torch.autograd.grad(1.5 * (a / a.sum(-1, keepdim=True) if renorm else a), x, up.double())
    s, a = s.detach(), a.detach()
    total = a.sum(-1, keepdim=True) if renorm else torch.ones_like(a[:, :1])
    mag = 1.5 * (up.abs().amax(-1, keepdim=True) * 2 / total) * s
    if scoring == "sigmoid":
        mag = mag * torch.zeros_like(s).scatter(-1, ids.long(), 1.0)
    u = torch.finfo(logits.dtype).eps / 2
    assert d.dtype == logits.dtype
    assert ((d.double() - want).abs() <= want.abs() * u + mag * 2.0 ** -20 + torch.finfo(logits.dtype).smallest_normal * u * 2).all()


def test_gradient_against_differences(dev):
    from lockstep_amd.experts import route
    for scoring in ("softmax", "sigmoid"):
        logits = _logits(dev, 3, 16, "f32", 1)
        up = torch.randn((3, 4), generator=torch.Generator(device=dev).manual_seed(2), device=dev)
        lg = logits.clone().requires_grad_(True)
        w, ids = route(lg, 4, scoring=scoring)
        d, = torch.autograd.grad(w, lg, up)
        for r, e in ((0, int(ids[0, 0])), (1, int(ids[1, 3])), (2, 7)):
            step = torch.zeros_like(logits)
            step[r, e] = 2.0 ** -8
            (p, pi), (q, qi) = route(logits + step, 4, scoring=scoring), route(logits - step, 4, scoring=scoring)
            if torch.equal(pi, ids) and torch.equal(qi, ids):
                assert abs(float(((p - q).double() * up).sum()) / 2.0 ** -7 - float(d[r, e])) < 1e-3


def test_shapes_strides_and_streams(dev):
    from lockstep_amd.experts import route
    base = _logits(dev, 12, 70, "f32", 3)
    want = route(base[:, :64].contiguous(), 4)
    for x in (base[:, :64], base[:, :64].t().contiguous().t()):
        got = route(x, 4)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    got = route(base[:, :64].unflatten(0, (3, 4)), 4, mask=torch.ones((3, 4), dtype=torch.bool, device=dev))
    assert got[0].shape == (3, 4, 4) and torch.equal(got[1].flatten(0, 1), want[1])
    assert route(base[0, :64], 4)[1].shape == (4,)
    assert route(base[:0, :64], 4)[1].shape == (0, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = route(base[:, :64], 4)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


# ---------------------------------------------------------------- dispatch
@pytest.mark.parametrize("T,k,E", [(0, 4, 8), (1, 1, 1), (1, 8, 256), (64, 8, 128), (65, 3, 60), (700, 6, 64), (1024, 4, 1024),
                                   (1025, 4, 7), (5000, 8, 129), (40000, 2, 256)])
def test_dispatch(dev, T, k, E):
    from lockstep_amd.experts import dispatch
    ids = torch.randint(-3, E + 2, (T, k), generator=torch.Generator(device=dev).manual_seed(T), device=dev, dtype=torch.int32)
    ids[T // 2:T // 2 + 20] = E // 2                     # a run of one expert
    d = dispatch(ids, E)
    flat = ids.flatten()
    key, order = torch.sort(torch.where((flat >= 0) & (flat < E), flat, E), stable=True)
    assert torch.equal(d.order, order.to(torch.int32))
    assert torch.equal(d.offsets, torch.searchsorted(key, torch.arange(E + 1, device=dev, dtype=torch.int32)).to(torch.int32))


def test_dispatch_of_extreme_ids_and_one_expert(dev):
    from lockstep_amd.experts import dispatch
    ids = torch.tensor([[2 ** 31 - 1, -2 ** 31], [3, 3], [-1, 4]], dtype=torch.int32, device=dev)
    d = dispatch(ids, 4)
    assert d.offsets.tolist() == [0, 0, 0, 0, 2] and d.order.tolist() == [2, 3, 0, 1, 4, 5]
    same = torch.zeros((9000, 1), dtype=torch.int32, device=dev)
    d = dispatch(same, 3)
    assert torch.equal(d.order.long(), torch.arange(9000, device=dev)) and d.offsets.tolist() == [0, 9000, 9000, 9000]
    t = ids.t().contiguous().t()                          # strides
    assert dispatch(t, 4).order.tolist() == [2, 3, 0, 1, 4, 5]


def test_dispatch_replayed(dev):
    from lockstep_amd.experts import dispatch
    ids = torch.zeros((3000, 4), dtype=torch.int32, device=dev)
    dispatch(ids, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = dispatch(ids, 64)
    for k in range(3):
        ids.random_(0, 64, generator=torch.Generator(device=dev).manual_seed(k))
        graph.replay()
        torch.cuda.synchronize()
        e = dispatch(ids, 64)
        assert torch.equal(d.order, e.order) and torch.equal(d.offsets, e.offsets)

"""The norm, the router and the experts' products: the native forms against the
Python path, at the borders of the kernels' forms, several at once, captured and
replayed with their backward passes.  Bounds as in test_gpu_norm, test_gpu_route
and test_gpu_experts."""

import threading

import pytest
import torch

from lockstep_amd import _capi as C

from . import test_gpu_experts as experts_tests
from . import test_gpu_norm as norm_tests
from . import test_gpu_route as route_tests
from .test_fast_calls import Declines, Recorder, Sub, _run_with, _same

NAMES = ("rms_norm", "route", "dispatch", "expert_gated", "expert_combine")


def test_other_forms_are_left_to_the_python_path():
    """CPU tensors, subclasses, other types and argument counts."""
    x = torch.zeros((2, 64))
    for bad in (x, x.as_subclass(Sub), None, 3, [x]):
        assert C.fast.rms_norm(bad, bad, None, 1e-6, False) is None
        assert C.fast.route(bad, 2, None, "softmax", 1, 1, True, 1.0, None) is None
        assert C.fast.dispatch(bad, 4) is None
        assert C.fast.expert_gated(bad, bad, bad, bad, (bad, bad, bad)) is None
        assert C.fast.expert_combine(bad, bad, bad, bad, (bad, bad, bad), bad, torch.bfloat16) is None
    for name in NAMES:
        assert getattr(C.fast, name)() is None and getattr(C.fast, name)(x) is None


def _state(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    T, D, F, E, k = 40, 256, 64, 8, 2
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    x, r, w = rnd(T, D).bfloat16(), rnd(T, D).bfloat16(), rnd(D).bfloat16()
    x8, xs = experts_tests._rows(dev, (T, D), 1)
    h8, hs = experts_tests._rows(dev, (T, k, F), 2)
    h8, hs = torch.cat([h8.view(torch.uint8)] * 2, -1).view(h8.dtype), torch.cat([hs] * 2, -1)
    w13, s13 = experts_tests._weights(dev, E, 2 * F, D, 3)
    w2, s2 = experts_tests._weights(dev, E, 96, 2 * F, 4)
    ids = experts_tests._ids(dev, T, k, E, 5, 0.1)
    return x, r, w, rnd(T, E), 0.1 * rnd(E), ids, x8, xs, w13, s13, h8, hs, w2, s2, torch.rand((T, k), generator=g, device=dev)


def _forms(dev):
    """(call, native function, whether it takes the call)"""
    from lockstep_amd import experts
    from lockstep_amd.norm import add_rms_norm
    x, r, w, l, b, ids, x8, xs, w13, s13, h8, hs, w2, s2, rw = _state(dev)
    mask = torch.arange(40, device=dev) % 5 > 0
    d = experts.dispatch(ids, 8)
    up = torch.randn_like(x)

    def norm_grads(x, w, r=None, both=True, **kw):
        t = [v.detach().clone().requires_grad_(True) for v in ((x, w) if r is None else (x, w, r))]
        o = add_rms_norm(*t, **kw)
        o = (o,) if isinstance(o, torch.Tensor) else o
        o = o[:1 if r is None or not both else 2]
        return (*(v.detach() for v in o), *torch.autograd.grad(o, t, (up,) * len(o), allow_unused=True))

    def route_grads(l, k, **kw):
        t = l.detach().clone().requires_grad_(True)
        wt, i = experts.route(t, k, **kw)
        return wt.detach(), i, *torch.autograd.grad(wt.square().sum(), t)
    wide = torch.zeros((40, 300), device=dev).bfloat16()
    wide[:, :256] = x
    return [
        (lambda: add_rms_norm(x, w), "rms_norm", True), (lambda: add_rms_norm(x, w.float(), r, eps=1e-3), "rms_norm", True),
        (lambda: add_rms_norm(x, w, r, mxfp8=True), "rms_norm", True), (lambda: norm_grads(x, w), "rms_norm", True),
        (lambda: norm_grads(x, w, r), "rms_norm", True), (lambda: norm_grads(x, w.float(), r, mxfp8=True), "rms_norm", True),
        (lambda: norm_grads(x, w, r, both=False), "rms_norm", True),
        (lambda: add_rms_norm(wide[:, :256], w), "rms_norm", False), (lambda: add_rms_norm(x[:0], w), "rms_norm", False),
        (lambda: add_rms_norm(x, w, eps=0), "rms_norm", False),
        (lambda: experts.route(l, 2), "route", True), (lambda: experts.route(l, 3, bias=b, scoring="sigmoid", groups=4, top_groups=2), "route", True),
        (lambda: experts.route(l.bfloat16(), 2, mask=mask, renormalize=False, scale=2.5), "route", True),
        (lambda: route_grads(l, 3), "route", True), (lambda: route_grads(l.half(), 2, mask=mask, bias=b, scoring="sigmoid"), "route", True),
        (lambda: experts.route(l.t().contiguous().t(), 2), "route", False), (lambda: experts.route(l, 2, scale=1), "route", False),
        (lambda: tuple(experts.dispatch(ids, 8)), "dispatch", True), (lambda: tuple(experts.dispatch(ids[:0], 8)), "dispatch", False),
        (lambda: experts.expert_gated(x8, xs, w13, s13, d), "expert_gated", True),
        (lambda: experts.expert_gated(x8.view(torch.uint8), xs, w13, s13, d), "expert_gated", True),
        (lambda: experts.expert_gated(x8, xs, w13, s13.transpose(1, 2).contiguous().transpose(1, 2), d), "expert_gated", False),
        (lambda: (experts.expert_combine(h8, hs, w2, s2, d, rw),), "expert_combine", True),
        (lambda: (experts.expert_combine(h8, hs, w2, s2, d, rw, torch.float32),), "expert_combine", True),
        (lambda: (experts.expert_combine(h8, hs, w2, s2, d, rw.t().contiguous().t()),), "expert_combine", False),
    ]


@pytest.mark.gpu
def test_the_plain_forms_are_native(dev, monkeypatch):
    for i, (call, name, native) in enumerate(_forms(dev)):
        rec = Recorder(C.fast)
        got = _run_with(monkeypatch, C, rec, call)
        assert [t for t in rec.took if t[0] != "captures"] == [(name, native)], (i, rec.took)
        assert _same(got, _run_with(monkeypatch, C, Declines(), call)), i


@pytest.mark.gpu
def test_calls_under_modes_and_transforms_take_the_python_path(dev, monkeypatch):
    """As for the other calls: both paths raise the same, and none is native."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from lockstep_amd import experts
    from lockstep_amd.norm import add_rms_norm
    x, r, w, l, b, ids, x8, xs, w13, s13, h8, hs, w2, s2, rw = _state(dev)
    d = experts.dispatch(ids, 8)
    natives = [lambda: C.fast.rms_norm(x, w, r, 1e-6, False), lambda: C.fast.route(l, 2, None, "softmax", 1, 1, True, 1.0, None),
               lambda: C.fast.dispatch(ids, 8), lambda: C.fast.expert_gated(x8, xs, w13, s13, d),
               lambda: C.fast.expert_combine(h8, hs, w2, s2, d, rw, torch.bfloat16)]
    calls = [lambda: add_rms_norm(x, w, r)[0], lambda: experts.route(l, 2)[0], lambda: experts.dispatch(ids, 8).order,
             lambda: experts.expert_gated(x8, xs, w13, s13, d)[1], lambda: experts.expert_combine(h8, hs, w2, s2, d, rw)]
    took = []
    for native, call in zip(natives, calls):
        def fake(native=native, call=call):
            with FakeTensorMode(allow_non_fake_inputs=True):
                took.append(native())
                return call()

        def grad(native=native, call=call):
            def f(s):
                took.append(native())
                return (call().float() * s).sum()
            return torch.func.grad(f)(torch.ones((), device=dev))
        for f in (fake, grad):
            errors = []
            for fast in (C.fast, Declines()):
                try:
                    _run_with(monkeypatch, C, fast, f)
                    errors.append(None)
                except Exception as e:  # noqa: BLE001
                    errors.append((type(e), str(e)))
            assert errors[0] == errors[1]
        assert native() is not None
    assert len(took) == 20 and all(t is None for t in took)


@pytest.mark.gpu
def test_traced_and_forward_mode_calls_are_refused(dev):
    import torch.autograd.forward_ad as fw

    from lockstep_amd import experts
    from lockstep_amd.norm import add_rms_norm
    x, r, w, l, b, ids, x8, xs, w13, s13, h8, hs, w2, s2, rw = _state(dev)
    d = experts.dispatch(ids, 8)
    for f, t in ((lambda a: add_rms_norm(a, w, r), x), (lambda a: experts.route(a, 2), l), (lambda a: tuple(experts.dispatch(a, 8)), ids),
                 (lambda a: experts.expert_gated(x8, a, w13, s13, d), xs), (lambda a: experts.expert_combine(h8, hs, w2, s2, d, a), rw)):
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(f, (t,), check_trace=False)
        f(t)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: add_rms_norm(dual(x), w, r), lambda: add_rms_norm(x, dual(w), r), lambda: add_rms_norm(x, w, dual(r)),
                  lambda: experts.route(dual(l), 2)):
            with pytest.raises(NotImplementedError, match="forward mode"):
                f()


# rows and dims on both sides of each form's border
@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(2047, 1024), (2048, 1016), (512, 4096), (513, 4088), (256, 8192), (257, 8184), (4097, 4104), (3, 8200), (3, 16384),
                                 (3, 16392)])
def test_norm_forms(dev, T, D):
    norm_tests.test_forward(dev, "bf16", T, D, True)
    norm_tests.test_forward(dev, "f32", T, D, False)
    if D % 32 == 0:
        norm_tests.test_mxfp8(dev, "f16", T, D)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(9, 2056), (1100, 4096), (5, 4104), (1030, 8192), (1030, 8200), (7, 16384), (3, 16392)])
def test_norm_backward_forms(dev, T, D):
    norm_tests.test_gradients(dev, "bf16", T, D, True)
    norm_tests.test_gradients(dev, "f32", T, D, False)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [128, 129, 4096, 4097])
@pytest.mark.parametrize("E,k,groups,top", [(256, 8, 8, 4), (256, 16, 1, 1), (96, 9, 16, 5), (250, 7, 1, 1), (16, 16, 1, 1), (17, 17, 1, 1)])
def test_route_forms(dev, T, E, k, groups, top):
    route_tests.test_choice_and_weights(dev, "f32", T, E, k, groups, top, "sigmoid", True)
    route_tests.test_choice_and_weights(dev, "bf16", T, E, k, groups, top, "softmax", True)
    route_tests.test_choice_and_weights(dev, "f32", T, E, k, groups, top, "softmax", False)


@pytest.mark.gpu
def test_gradients_are_leaves_own(dev):
    """x and the residual get one gradient, in memory of their own."""
    from lockstep_amd.norm import add_rms_norm
    x, r, w = (t.requires_grad_(True) for t in norm_tests._inputs(dev, 5, 64, torch.float32, 1))
    y, h = add_rms_norm(x, w, r)
    (y.sum() + h.square().sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    want = x.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, want)


@pytest.mark.gpu
def test_training_pass_captured_and_replayed(dev):
    """Forward and backward in one graph, twice, replayed in turn, against eager passes."""
    from lockstep_amd import experts
    from lockstep_amd.norm import add_rms_norm
    T, D, E = 70, 256, 32
    x, r, w = norm_tests._inputs(dev, T, D, torch.bfloat16, 1)
    router = (0.1 * torch.randn((E, D), generator=torch.Generator(device=dev).manual_seed(2), device=dev)).bfloat16()
    leaves = [t.requires_grad_(True) for t in (x, w, r, router)]

    def step():
        y, h = add_rms_norm(x, w, r)
        wt, ids = experts.route(y @ router.t(), 4, scoring="sigmoid")
        loss = (wt * torch.arange(1, 5, device=dev)).sum() + h.float().square().mean()
        return [wt.detach(), ids, *torch.autograd.grad(loss, leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [], []
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.synchronize()
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            held.append(step())
    for i in range(4):
        with torch.no_grad():
            x.normal_(generator=torch.Generator(device=dev).manual_seed(i))
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(p, q) for p, q in zip(held[i % 2], want)), i
        del want


@pytest.mark.gpu
def test_capture_after_a_warm_up_on_another_stream(dev):
    """The usual recipe: a warm-up on a side stream, whose outputs are still held, then
    the capture on the graph's own."""
    from lockstep_amd import experts
    from lockstep_amd.norm import add_rms_norm
    x, r, w = (t.requires_grad_(True) for t in norm_tests._inputs(dev, 33, 64, torch.float32, 4))

    def step():
        y, h = add_rms_norm(x, w, r)
        wt, ids = experts.route(y, 4)
        return (wt * torch.arange(1, 5, device=dev)).sum() + h.square().mean()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            loss = step()
            grads = torch.autograd.grad(loss, (x, w, r))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
        held_grads = torch.autograd.grad(held, (x, w, r))
    del loss, grads
    for i in range(3):
        with torch.no_grad():
            x.normal_(generator=torch.Generator(device=dev).manual_seed(i))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = torch.autograd.grad(step(), (x, w, r))
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held_grads, want))


@pytest.mark.gpu
def test_threads_and_streams_at_once(dev):
    """Four threads, a stream each, one run of the operators: as when alone."""
    from lockstep_amd import experts, fp4
    from lockstep_amd.norm import add_rms_norm
    T, D, F, E, k = 5000, 256, 128, 16, 2
    g = torch.Generator(device=dev).manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    xs, nw, router = [rnd(T, D).bfloat16() for _ in range(4)], rnd(D).bfloat16(), 0.1 * rnd(E, D).bfloat16()
    w13, s13 = fp4.quantize_pack_mxfp4((0.06 * rnd(E, 2 * F, D)).bfloat16())
    w2, s2 = fp4.quantize_pack_mxfp4((0.1 * rnd(E, D, F)).bfloat16())

    def layer(x):
        y, x8, xsc = add_rms_norm(x, nw, mxfp8=True)
        wt, ids = experts.route(y @ router.t(), k)
        d = experts.dispatch(ids, E)
        a, s = experts.expert_gated(x8, xsc, w13, s13, d)
        return experts.expert_combine(a, s, w2, s2, d, wt)
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[i] = layer(xs[i])
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,F", [(6, 256, 64), (200, 512, 128)])
def test_one_expert_twice_for_a_token_and_padding(dev, T, K, F):
    """A token may name an expert twice: each slot is a pair of its own.  Padded
    tokens' rows, of any contents, change nothing, and come out as zeros."""
    from lockstep_amd import experts
    E, k = 3, 4
    x, xs = experts_tests._rows(dev, (T, K), 1)
    w, ws = experts_tests._weights(dev, E, 2 * F, K, 2)
    w2, w2s = experts_tests._weights(dev, E, 96, 2 * F, 3)
    ids = torch.tensor([[1, 1, 2, 1]], dtype=torch.int32, device=dev).expand(T, k).contiguous()
    ids[T // 2:] = -1
    x2, xs2 = x.clone(), xs.clone()
    x2.view(torch.uint8)[T // 2:] = 0x7F     # NaN
    xs2[T // 2:] = 255
    d = experts.dispatch(ids, E)
    h, hs = experts.expert_gated(x2, xs2, w, ws, d)
    one, ones = experts.expert_gated(x[:T // 2], xs[:T // 2], w, ws, experts.dispatch(ids[:T // 2], E))
    same = lambda p, q: torch.equal(p.view(torch.uint8), q.view(torch.uint8))  # noqa: E731
    assert same(h[:, 0].contiguous(), h[:, 1].contiguous()) and same(h[:, 0].contiguous(), h[:, 3].contiguous())
    assert (h[T // 2:].view(torch.uint8) == 0).all() and (hs[T // 2:] == 127).all()
    # alone they may take another form of the kernel: within a code of the formula's
    p, q = (experts_tests._values8(*t) for t in ((h[:T // 2], hs[:T // 2]), (one, ones)))
    assert ((p - q).abs() <= q.abs() * 2.0 ** -3 + 2.0 ** -9 * torch.exp2(ones.double() - 127).repeat_interleave(32, -1)).all()
    h2 = torch.cat([h.view(torch.uint8)] * 2, -1).view(h.dtype)
    rw = torch.rand((T, k), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    rw[T // 2:] = float("nan")
    y = experts.expert_combine(h2, torch.cat([hs] * 2, -1), w2, w2s, d, rw)
    assert (y[T // 2:] == 0).all() and torch.isfinite(y.float()).all()


@pytest.mark.gpu
def test_weights_and_rows_beyond_32_bits(dev):
    """Experts whose weights, and pairs whose rows, lie past 2^32 bytes."""
    from lockstep_amd import experts
    E, N, K = 36, 4096, 2 ** 16
    w = torch.zeros((E, N, K // 2), dtype=torch.uint8, device=dev)          # 4.8 GB
    ws = torch.full((E, N, K // 32), 127, dtype=torch.uint8, device=dev)
    w[E - 1, :, K // 2 - 1] = 0x20                                          # one in the last column
    w[0, :, 0] = 0x02
    T = 70000                                                               # 4.6 GB of rows
    x = torch.zeros((T, 1, K), dtype=torch.uint8, device=dev)
    xs = torch.full((T, 1, K // 32), 127, dtype=torch.uint8, device=dev)
    n = torch.arange(T, device=dev)
    x[:, 0, K - 1] = (0x38 + n % 8).to(torch.uint8)                         # 1 + (n % 8) / 8
    x[:, 0, 0] = 0x40
    ids = torch.full((T, 1), E - 1, dtype=torch.int32, device=dev)
    ids[::7] = 0
    d = experts.dispatch(ids, E)
    y = experts.expert_combine(x.view(torch.float8_e4m3fn), xs, w, ws, d, torch.ones((T, 1), device=dev), torch.float32)
    want = torch.where(n % 7 == 0, 2.0, 1 + (n % 8) / 8.0)
    assert torch.equal(y, want[:, None].expand(T, N))
    few = torch.tensor([[T - 1], [3]], device=dev)
    y = experts.expert_combine(x.view(torch.float8_e4m3fn)[-2:].contiguous(), xs[-2:].contiguous(), w, ws,
                               experts.dispatch(ids[-2:].contiguous(), E), torch.ones((2, 1), device=dev), torch.float32)
    assert torch.equal(y, want[-2:, None].expand(2, N)) and few.numel() == 2


@pytest.mark.gpu
def test_leaves_of_another_streams_graph_are_told(dev):
    """The check that a captured call makes, with the capture's part played by the
    host: only a tensor whose graph, still alive, is the default stream's is refused."""
    x, r, w = (t.requires_grad_(True) for t in norm_tests._inputs(dev, 6, 64, torch.float32, 3))
    from lockstep_amd.norm import add_rms_norm
    side = torch.cuda.Stream()
    eager = add_rms_norm(x, w)
    side.wait_stream(torch.cuda.current_stream())
    C.fast.captures((x, w, r, x * 2), True)
    with torch.cuda.stream(side):
        C.fast.captures((r, x.detach()), True)            # no graph of r
        for t in (x, w, eager):
            C.fast.captures((t,), False)
            C.fast.captures((t,), None)                   # nothing is captured here
            with pytest.raises(RuntimeError, match="on the default stream is alive"):
                C.fast.captures((r, t), True)
        del eager, t
        C.fast.captures((x, w), True)
        y = add_rms_norm(x, w)
        C.fast.captures((x, w, y), True)
    side.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        C.fast.captures((x, w, y), True)                  # a stream that can join the capture


@pytest.mark.gpu
@pytest.mark.skip(reason="ended the process in capture_end when the refusal came from the backward pass, for a cause not shown; "
                         "the refusal now comes before anything is captured (the test above)")
def test_a_capture_while_an_eager_graph_lives(dev):
    """Is refused, and the eager graph's own backward pass goes on."""
    from lockstep_amd import experts
    from lockstep_amd.norm import add_rms_norm
    x, r, w = (t.requires_grad_(True) for t in norm_tests._inputs(dev, 6, 64, torch.float32, 3))
    l = torch.randn((6, 8), generator=torch.Generator(device=dev).manual_seed(1), device=dev, requires_grad=True)
    for f, t in ((lambda: add_rms_norm(x, w, r)[0], (x, w, r)), (lambda: experts.route(l, 2)[0], (l,))):
        eager = f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                torch.autograd.grad(f().sum(), t)
        torch.cuda.synchronize()
        assert all(torch.isfinite(g).all() for g in torch.autograd.grad(eager.sum(), t))
        del eager


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [100, 5000])
def test_groups_whose_ranks_cancel_or_logits_are_large(dev, T, scoring):
    """A group's two largest ranks of +-1000 add up to little, with the rounding of
    1000; a softmax of logits near 3000 depends on what 32 bits hold of them."""
    E, k, G = 128, 4, 16
    g = torch.Generator(device=dev).manual_seed(T)
    logits = torch.randn((T, E), generator=g, device=dev)
    bias = torch.full((E,), -1000.0, device=dev)
    bias[::8] = 1000.0
    bias += (torch.randint(-4, 5, (E,), generator=g, device=dev) * 2.0 ** -13)
    from lockstep_amd.experts import route
    w, ids = route(logits, k, bias=bias, scoring=scoring, groups=G, top_groups=3)
    _, at = route_tests._route64(logits, k, bias, scoring, G, 3, True, 1.0)
    assert torch.equal(ids.long(), at)
    big = (2990 + torch.randint(0, 40, (T, E), generator=g, device=dev) * 2.0 ** -12).float()
    w, ids = route(big, k, scoring="softmax", groups=G, top_groups=3)
    want, at = route_tests._route64(big, k, None, "softmax", G, 3, True, 1.0)
    assert torch.equal(ids.long(), at) and ((w.double() - want).abs() <= want * 2.0 ** -20).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E", [(1024, 1, 32), (1025, 1, 7), (1024, 2, 60), (683, 3, 1024), (8192, 8, 32), (65537, 1, 256), (262144, 8, 64)])
def test_dispatch_forms(dev, T, k, E):
    route_tests.test_dispatch(dev, T, k, E)


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes(dev):
    """Past 2^21 rows of the norm and 2^22 of the router: rows near each border as when alone."""
    from lockstep_amd.experts import route
    from lockstep_amd.norm import add_rms_norm
    T = 2 ** 22 + 5
    g = torch.Generator(device=dev).manual_seed(0)
    x, r = (torch.randn((T, 32), generator=g, device=dev).bfloat16() for _ in range(2))
    w = torch.randn(32, generator=g, device=dev).bfloat16()
    got = add_rms_norm(x, w, r, mxfp8=True)
    part = [slice(a, a + 9) for a in (0, 2 ** 21 - 4, 2 ** 22 - 4)]
    for p in part:
        want = add_rms_norm(x[p].contiguous(), w, r[p].contiguous(), mxfp8=True)
        assert all(torch.equal(u[p].view(torch.uint8), v.view(torch.uint8)) for u, v in zip(got, want))
    l = torch.randn((T, 5), generator=g, device=dev)
    mask = torch.rand(T, generator=g, device=dev) < 0.9
    up = torch.randn((T, 2), generator=g, device=dev)

    def both(p):
        t = l[p].clone().requires_grad_(True)
        wt, ids = route(t, 2, mask=mask[p].contiguous())
        return wt.detach(), ids, torch.autograd.grad(wt, t, up[p].contiguous())[0]
    got = both(slice(None))
    for p in part:
        assert all(torch.equal(u[p], v) for u, v in zip(got, both(p)))


@pytest.mark.gpu
def test_empty_rows_are_refused_and_no_rows_are_not(dev):
    from lockstep_amd.experts import route
    from lockstep_amd.norm import add_rms_norm
    with pytest.raises(AssertionError, match="at least 1"):
        add_rms_norm(torch.zeros((3, 0), device=dev), torch.zeros(0, device=dev))
    with pytest.raises(AssertionError, match="must be"):
        route(torch.zeros((3, 0), device=dev), 1)
    x, w = (torch.zeros(s, device=dev, requires_grad=True) for s in ((0, 64), (64,)))
    y, h = add_rms_norm(x, w, x)
    gx, gw = torch.autograd.grad(y.sum() + h.sum(), (x, w))
    assert gx.shape == (0, 64) and torch.equal(gw, torch.zeros_like(w))
    l = torch.zeros((0, 8), device=dev, requires_grad=True)
    wt, ids = route(l, 2)
    assert ids.shape == (0, 2) and torch.autograd.grad(wt.sum(), l)[0].shape == (0, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("E,K,F,pairs", [(1, 512, 32, 3000), (3, 512, 160, 2000), (2, 1152, 96, 800), (9, 768, 128, 4000)])
def test_uneven_experts_and_borders_of_tiles(dev, E, K, F, pairs):
    """Experts without a pair, with one, with a tile's and one more; rows of W past a tile's end."""
    from lockstep_amd import experts
    g = torch.Generator(device=dev).manual_seed(pairs)
    x, xs = experts_tests._rows(dev, (pairs, K), 1)
    w, ws = experts_tests._weights(dev, E, 2 * F, K, 2)
    ids = torch.full((pairs, 1), E - 1, dtype=torch.int32, device=dev)
    if E > 1:
        ids[:257] = 0
    if E > 3:
        ids[300] = 1
        ids[400:528] = 3
        ids[600:1112] = 5
    ids = ids[torch.randperm(pairs, generator=g, device=dev)].contiguous()
    d = experts.dispatch(ids, E)
    h, hs = experts.expert_gated(x, xs, w, ws, d)
    out, mag = experts_tests._products(experts_tests._values8(x, xs), ids, w, ws, False)
    gate, up = out.chunk(2, -1)
    dg, du = (mag * experts_tests.IN_BLOCK).chunk(2, -1)
    want = gate * torch.sigmoid(gate) * up
    err = 1.1 * dg * (up.abs() + du) + (gate * torch.sigmoid(gate)).abs() * du + want.abs() * 2.0 ** -18
    step = torch.exp2(hs.double() - 127).repeat_interleave(32, -1) * 2.0 ** -10
    assert ((experts_tests._values8(h, hs) - want).abs() <= err * (1 + 2.0 ** -4) + want.abs() * 2.0 ** -4 + step).all()
    x3, xs3 = x[:, None], xs[:, None]
    for dt in (torch.bfloat16, torch.float16):
        y = experts.expert_combine(x3.contiguous(), xs3.contiguous(), w, ws, d, torch.ones((pairs, 1), device=dev), dt)
        assert ((y.double() - out[:, 0]).abs() <= out[:, 0].abs() * torch.finfo(dt).eps / 2 + mag[:, 0] * (experts_tests.IN_BLOCK + 2.0 ** -11)
                ).all()

"""The native forms of the attention and cache calls: the plain ones are taken, and
give the Python path's bits; others are left to it."""

import pytest
import torch

from lockstep_amd import _capi as C

from .test_fast_calls import Declines, Recorder, Sub, _run_with, _same

NAMES = ("attention", "kv_append", "kv_attend", "kv_evict")


def test_other_forms_are_left_to_the_python_path():
    """CPU tensors, subclasses, other types and argument counts."""
    x = torch.zeros((1, 2, 2, 64), dtype=torch.bfloat16)
    pages = tuple(torch.zeros((2, 2, 16, n), dtype=torch.uint8) for n in (32, 2, 32, 2))
    t, n, w = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros((1, 2, 16))
    for bad in (x, x.as_subclass(Sub), None, 3, [x]):
        assert C.fast.attention(bad, bad, bad, None, None, 0, None) is None
        assert C.fast.kv_append(pages, bad, bad, t, n, None, False) is None
        assert C.fast.kv_attend(bad, pages, t, n, None, 0, None, None) is None
    assert C.fast.kv_attend(x, None, t, n, None, 0, None, None) is None
    assert C.fast.kv_evict(pages, t, n, w, 4, t, 0, 0) is None
    for name in NAMES:
        assert getattr(C.fast, name)() is None and getattr(C.fast, name)(x) is None


def state(dev, dt=torch.bfloat16):
    from lockstep_amd import kv_cache as kc
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, device=dev).to(dt)  # noqa: E731
    q, k, v = r(2, 40, 6, 64), r(2, 40, 2, 64), r(2, 40, 2, 64)
    pages = kc.new_pages(12, 2, 64, 16, device=dev)
    table = torch.arange(6, dtype=torch.int32, device=dev).view(2, 3)
    lengths = torch.full((2,), 40, dtype=torch.int32, device=dev)
    out = torch.arange(6, 12, dtype=torch.int32, device=dev).view(2, 3)
    w = torch.rand((2, 2, 48), generator=g, device=dev)
    kc.append(pages, k, v, table, lengths)
    return q, k, v, pages, table, lengths, out, w


def forms(dev, dt):
    """(call, native function, whether it takes the call)"""
    from lockstep_amd import kv_cache as kc
    from lockstep_amd.attention import sink_window_attention as f
    q, k, v, pages, table, lengths, out, w = state(dev, dt)
    off = torch.tensor([0, 30, 80], dtype=torch.int32, device=dev)
    qp, kp, vp = (t.flatten(0, 1) for t in (q, k, v))
    odd = torch.nn.functional.pad(k, (1, 0))[..., 1:]            # not 16-byte aligned
    copy = lambda: kc.Pages(*(t.clone() for t in pages))  # noqa: E731

    def grads(*x, **kw):
        x = [t.clone().requires_grad_(True) for t in x]
        o = f(*x, **kw)
        return (o.detach(), *torch.autograd.grad(o.float().square().sum(), x))

    def append(k, v, **kw):
        p = copy()
        return (kc.append(p, k, v, table, lengths, **kw) or ()) + tuple(p)

    def attend(q, weights=None, **kw):
        weights = None if weights is None else weights.clone()
        o = kc.attend(q, pages, table, lengths, weights=weights, **kw)
        return (o,) if weights is None else (o, weights)

    def evict(w, keep, **kw):
        p = copy()
        return (*kc.evict(p, table, lengths, w, keep, out, **kw), *p)
    return [
        (lambda: f(q, k, v), "attention", True), (lambda: f(q, k, v, window=9, sinks=2, scale=0.2), "attention", True),
        (lambda: f(qp, kp, vp, offsets=off), "attention", True), (lambda: grads(q, k, v, window=9), "attention", True),
        (lambda: grads(qp, kp, vp, offsets=off, sinks=1, window=20), "attention", True),
        (lambda: f(q, odd, v), "attention", False), (lambda: f(q, k, v, scale=1), "attention", False),
        (lambda: f(q[:, :0], k, v), "attention", False),
        (lambda: append(k, v), "kv_append", True), (lambda: append(k, v, values=True), "kv_append", True),
        (lambda: append(kp, vp, offsets=torch.tensor([0, 40, 80], dtype=torch.int32, device=dev)), "kv_append", True),
        (lambda: append(odd, v), "kv_append", False), (lambda: append(k[:, :0], v[:, :0], values=True), "kv_append", False),
        (lambda: attend(q[:, :1]), "kv_attend", True), (lambda: attend(q, w, window=11, sinks=3), "kv_attend", True),
        (lambda: attend(q, w), "kv_attend", True), (lambda: attend(odd), "kv_attend", False),
        (lambda: evict(w, 20, sinks=1, recent=4), "kv_evict", True), (lambda: evict(w, 48), "kv_evict", True),
    ]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_the_plain_forms_are_native(dt, dev, monkeypatch):
    for i, (call, name, native) in enumerate(forms(dev, dt)):
        rec = Recorder(C.fast)
        got = _run_with(monkeypatch, C, rec, call)
        assert rec.took == [(name, native)], (i, rec.took)
        assert _same(got, _run_with(monkeypatch, C, Declines(), call)), i


@pytest.mark.gpu
def test_calls_under_modes_and_transforms_take_the_python_path(dev, monkeypatch):
    """As for the other calls: both paths raise the same, and none is native."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from lockstep_amd import kv_cache as kc
    from lockstep_amd.attention import sink_window_attention
    q, k, v, pages, table, lengths, out, w = state(dev)
    natives = [lambda: C.fast.attention(q, k, v, None, None, 0, None),
               lambda: C.fast.kv_append(pages, k, v, table, lengths, None, True),
               lambda: C.fast.kv_attend(q, pages, table, lengths, None, 0, None, None),
               lambda: C.fast.kv_evict(pages, table, lengths, w, 20, out, 0, 0)]
    calls = [lambda: sink_window_attention(q, k, v), lambda: kc.append(pages, k, v, table, lengths, values=True)[0],
             lambda: kc.attend(q, pages, table, lengths), lambda: kc.evict(pages, table, lengths, w, 20, out)[1]]
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
    assert len(took) == 16 and all(r is None for r in took)


@pytest.mark.gpu
def test_errors_are_the_python_path_s(dev):
    """A call that the library refuses raises LsmxError from both paths."""
    from lockstep_amd.attention import sink_window_attention
    q, k, v, *_ = state(dev)
    for fast in (C.fast, Declines()):
        keep, C.fast = C.fast, fast
        try:
            with pytest.raises(C.LsmxError, match="scale"):
                sink_window_attention(q, k, v, scale=1e-60)     # 0 in fp32
        finally:
            C.fast = keep

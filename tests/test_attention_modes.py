"""The attention and cache calls under forward-mode derivatives and torch.jit.trace:
nothing is dropped without an error.  On the CPU with the kernels stubbed, which
is the Python path; on the GPU the native one."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from lockstep_amd import _capi as C
from lockstep_amd import kv_cache as kc
from lockstep_amd.attention import sink_window_attention


class Declines:
    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture
def stubs(monkeypatch):
    """CPU tensors pass, and no kernel is called."""
    monkeypatch.setattr(C, "fast", Declines())
    monkeypatch.setattr(C, "call", lambda *a: None)
    monkeypatch.setattr(C, "require_device", lambda *a: None)
    monkeypatch.setattr(C, "stream_of", lambda t: 0)


def _inputs(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    return [torch.randn((1, 9, h, 64), generator=g, device=dev).bfloat16() for h in (4, 2, 2)]


def _forward_mode(dev):
    for which in range(3):
        for grad in (False, True):
            x = [t.requires_grad_(grad) for t in _inputs(dev)]
            with fw.dual_level():
                x[which] = fw.make_dual(x[which].detach(), torch.ones_like(x[which]))
                for off in (None, torch.tensor([0, 9], dtype=torch.int32, device=dev)):
                    y = x if off is None else [t[0] for t in x]
                    with pytest.raises(NotImplementedError, match="forward mode"):
                        sink_window_attention(*y, offsets=off)
                    with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                        sink_window_attention(*y, offsets=off)
            # a level without a dual tensor changes nothing
            with fw.dual_level():
                assert sink_window_attention(*_inputs(dev)).shape == (1, 9, 4, 64)


def _trace(dev):
    q, k, v = _inputs(dev)
    pages = kc.new_pages(4, 2, 64, 16, device=dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    out = torch.ones((1, 1), dtype=torch.int32, device=dev)
    lengths = torch.full((1,), 9, dtype=torch.int32, device=dev)
    w = torch.zeros((1, 2, 16), device=dev)
    calls = [(lambda a: sink_window_attention(a, k, v), q), (lambda a: kc.attend(a, pages, table, lengths), q),
             (lambda a: kc.append(pages, a, v, table, lengths, values=True), k),
             (lambda a: kc.evict(pages, table, lengths, a, 8, out), w)]
    for f, x in calls:
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(f, (x,), check_trace=False)
        f(x)


def test_forward_mode_python(stubs):
    _forward_mode(torch.device("cpu"))


def test_trace_python(stubs):
    _trace(torch.device("cpu"))


@pytest.mark.gpu
def test_forward_mode_native(dev):
    _forward_mode(dev)


@pytest.mark.gpu
def test_trace_native(dev):
    _trace(dev)

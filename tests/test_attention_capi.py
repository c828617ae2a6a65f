"""CPU tests of the attention and cache entry points: bad arguments come back
as errors before a device is touched, at the C ABI and in Python, and their
kernels compile without scratch memory."""

import ctypes
import re
import subprocess

import pytest
import torch

from lockstep_amd import _capi as C

from .test_kernel_resources import CSRC, _hipcc

FAKE = 0x1000   # never dereferenced: validation fails first
I3 = ctypes.c_int64 * 3
BIG = 2 ** 62


def attention(**kw):
    a = C.Attention(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, C.BF16, 2, 16, 16, 4, 2, 64, I3(4096, 256, 64),
                    I3(2048, 128, 64), I3(2048, 128, 64), I3(4096, 256, 64), None, 0, 0, 0.125)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


ATTENTION = [
    (dict(dtype=C.F32), C.ERR_DTYPE), (dict(q_len=-1), C.ERR_SHAPE), (dict(batch=-1), C.ERR_SHAPE),
    (dict(heads=3), C.ERR_SHAPE), (dict(kv_heads=0), C.ERR_SHAPE), (dict(heads=0), C.ERR_SHAPE),
    (dict(head_dim=136), C.ERR_SHAPE), (dict(head_dim=12), C.ERR_SHAPE), (dict(head_dim=0), C.ERR_SHAPE),
    (dict(offsets=FAKE, k_len=15), C.ERR_SHAPE), (dict(window=-1), C.ERR_ARG), (dict(sinks=-1), C.ERR_ARG),
    (dict(scale=0.0), C.ERR_ARG), (dict(scale=float("nan")), C.ERR_ARG), (dict(scale=float("inf")), C.ERR_ARG),
    (dict(q_len=BIG), C.ERR_SHAPE), (dict(k_len=BIG), C.ERR_SHAPE), (dict(batch=BIG), C.ERR_SHAPE),
    (dict(q_len=2 ** 29), C.ERR_SHAPE), (dict(batch=2 ** 29), C.ERR_SHAPE),
    (dict(q=None), C.ERR_ARG), (dict(o=None), C.ERR_ARG), (dict(k=None), C.ERR_ARG), (dict(v=None), C.ERR_ARG),
    (dict(q=FAKE + 8), C.ERR_ALIGN), (dict(v=FAKE + 2), C.ERR_ALIGN), (dict(offsets=FAKE + 1), C.ERR_ALIGN),
    (dict(q_stride=I3(4096, 260, 64)), C.ERR_ALIGN), (dict(k_stride=I3(4096, 2 ** 22, 64)), C.ERR_SHAPE),
    (dict(v_stride=I3(4096, -64, 64)), C.ERR_SHAPE), (dict(q_stride=I3(4096, 256, -64)), C.ERR_SHAPE),
]


@pytest.mark.parametrize("change,code", ATTENTION)
def test_attention_refusals(change, code):
    lib, a, st = C.load(), attention(**change), I3(4096, 256, 64)
    assert lib.lsmx_attention_fwd(ctypes.byref(a), None) == code and "lsmx_attention_fwd" in C.last_error()
    assert lib.lsmx_attention_bwd(ctypes.byref(a), FAKE, ctypes.byref(st), FAKE, FAKE, FAKE, FAKE, BIG,
                                  None) == code
    assert lib.lsmx_attention_workspace(ctypes.byref(a)) == 0


def test_attention_backward_refusals():
    lib, st = C.load(), I3(4096, 256, 64)
    n = lib.lsmx_attention_workspace(ctypes.byref(attention()))
    assert n > 0

    def rc(a=None, d_o=FAKE, st=st, dq=FAKE, dk=FAKE, dv=FAKE, ws=FAKE, n=n):
        a = a or attention()
        return lib.lsmx_attention_bwd(ctypes.byref(a), d_o, ctypes.byref(st) if st else None, dq, dk, dv, ws, n, None)
    for bad in (dict(d_o=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(ws=None), dict(n=n - 1), dict(st=None),
                dict(a=attention(lse=None)), dict(a=attention(o_rest=None))):
        assert rc(**bad) == C.ERR_ARG, bad
    for bad in (dict(d_o=FAKE + 2), dict(dq=FAKE + 8), dict(ws=FAKE + 4), dict(st=I3(4096, 252, 64))):
        assert rc(**bad) == C.ERR_ALIGN, bad
    for bad in (dict(st=I3(0, 2 ** 22, 64)), dict(st=I3(0, 256, 2 ** 28)), dict(a=attention(q_stride=I3(0, 0, 2 ** 28)))):
        assert rc(**bad) == C.ERR_SHAPE, bad
    assert lib.lsmx_attention_bwd(None, FAKE, None, FAKE, FAKE, FAKE, FAKE, n, None) == C.ERR_ARG
    assert lib.lsmx_attention_fwd(None, None) == C.ERR_ARG


def test_attention_backward_of_tokens_in_no_sequence():
    """Packed without a sequence: the tokens' gradients are written (zeros), so lse
    and o_rest are read and must be there."""
    lib, st = C.load(), I3(0, 256, 64)
    for bad in (dict(lse=None), dict(o_rest=None)):
        a = attention(batch=0, offsets=FAKE, **bad)
        n = lib.lsmx_attention_workspace(ctypes.byref(a))
        assert lib.lsmx_attention_bwd(ctypes.byref(a), FAKE, ctypes.byref(st), FAKE, FAKE, FAKE, FAKE, n, None) == C.ERR_ARG
        assert "o_rest" in C.last_error()


def cache(**kw):
    c = C.KVCache(FAKE, FAKE, FAKE, FAKE, 8, 16, 2, 64, FAKE, FAKE, 2, 4)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


CACHE = [
    (dict(pages=-1), C.ERR_SHAPE), (dict(batch=-1), C.ERR_SHAPE), (dict(max_pages=-1), C.ERR_SHAPE),
    (dict(kv_heads=0), C.ERR_SHAPE), (dict(page=8), C.ERR_SHAPE), (dict(page=24), C.ERR_SHAPE),
    (dict(page=2048), C.ERR_SHAPE), (dict(head_dim=96), C.ERR_SHAPE), (dict(pages=BIG), C.ERR_SHAPE),
    (dict(max_pages=BIG), C.ERR_SHAPE), (dict(max_pages=2 ** 60), C.ERR_SHAPE), (dict(batch=BIG), C.ERR_SHAPE),
    (dict(kv_heads=2 ** 29, batch=2 ** 29), C.ERR_SHAPE), (dict(k_codes=None), C.ERR_ARG), (dict(v_scale=None), C.ERR_ARG),
    (dict(table=None), C.ERR_ARG), (dict(lengths=None), C.ERR_ARG), (dict(k_codes=FAKE + 8), C.ERR_ALIGN),
    (dict(table=FAKE + 2), C.ERR_ALIGN),
]


def _append(c, k=FAKE, ks=(128, 64), v=FAKE, vs=(128, 64), dtype=C.BF16, tokens=6, per=3, offsets=None, ko=None, vo=None):
    I2 = ctypes.c_int64 * 2
    ks, vs = I2(*ks), I2(*vs)
    return C.load().lsmx_kv_append(ctypes.byref(c) if c else None, k, ctypes.byref(ks), v, ctypes.byref(vs),
                                   dtype, tokens, per, offsets, ko, vo, None)


def _attend(c, q=FAKE, qs=(256, 256, 64), dtype=C.BF16, T=1, H=4, window=0, sinks=0, scale=0.125, o=FAKE, w=None, w_len=0,
            ws=FAKE, n=BIG):
    qs = I3(*qs)
    return C.load().lsmx_kv_attend(ctypes.byref(c) if c else None, q, ctypes.byref(qs), dtype, T, H, window, sinks,
                                   scale, o, w, w_len, ws, n, None)


def _evict(c, w=FAKE, w_len=64, keep=20, sinks=1, recent=2, out=FAKE, out_pages=2, index=FAKE, kept=FAKE, new=FAKE):
    return C.load().lsmx_kv_evict(ctypes.byref(c) if c else None, w, w_len, keep, sinks, recent, out, out_pages, index,
                                  kept, new, None)


@pytest.mark.parametrize("change,code", CACHE)
def test_cache_refusals(change, code):
    for call in (_append, _attend, _evict):
        assert call(cache(**change)) == code, call.__name__
    assert C.load().lsmx_kv_attend_workspace(ctypes.byref(cache(**change)), 1, 4, 0, 0, 1) == 0


def test_cache_call_refusals():
    for call in (_append, _attend, _evict):
        assert call(None) == C.ERR_ARG
    c = cache()
    for bad, code in ((dict(dtype=C.F32), C.ERR_DTYPE), (dict(tokens=-1, per=-1), C.ERR_SHAPE), (dict(tokens=5), C.ERR_SHAPE),
                      (dict(tokens=BIG), C.ERR_SHAPE), (dict(tokens=0, per=2 ** 63 - 1), C.ERR_SHAPE), (dict(k=None), C.ERR_ARG),
                      (dict(ko=FAKE), C.ERR_ARG), (dict(k=FAKE + 4), C.ERR_ALIGN), (dict(ks=(130, 64)), C.ERR_ALIGN),
                      (dict(vs=(128, 60)), C.ERR_ALIGN), (dict(offsets=FAKE + 2), C.ERR_ALIGN)):
        assert _append(c, **bad) == code, bad
    need = C.load().lsmx_kv_attend_workspace(ctypes.byref(c), 1, 4, 0, 0, 1)
    assert need > 0
    for bad, code in ((dict(dtype=C.F32), C.ERR_DTYPE), (dict(H=3), C.ERR_SHAPE), (dict(H=0), C.ERR_SHAPE),
                      (dict(T=-1), C.ERR_SHAPE), (dict(T=BIG), C.ERR_SHAPE), (dict(H=BIG), C.ERR_SHAPE),
                      (dict(window=-1), C.ERR_ARG), (dict(sinks=-1), C.ERR_ARG), (dict(scale=0.0), C.ERR_ARG),
                      (dict(scale=float("nan")), C.ERR_ARG), (dict(q=None), C.ERR_ARG), (dict(o=None), C.ERR_ARG),
                      (dict(w=FAKE, w_len=63), C.ERR_SHAPE), (dict(w=FAKE, w_len=64, n=need - 1), C.ERR_ARG),
                      (dict(w=FAKE, w_len=64, ws=None), C.ERR_ARG), (dict(w=FAKE + 2, w_len=64), C.ERR_ALIGN),
                      (dict(q=FAKE + 8), C.ERR_ALIGN), (dict(qs=(256, 256, 60)), C.ERR_ALIGN)):
        assert _attend(c, **bad) == code, bad
    for bad, code in ((dict(keep=0), C.ERR_ARG), (dict(keep=BIG), C.ERR_ARG), (dict(sinks=-1), C.ERR_ARG),
                      (dict(recent=-1), C.ERR_ARG), (dict(sinks=10, recent=11), C.ERR_ARG),
                      (dict(sinks=BIG, recent=BIG), C.ERR_ARG), (dict(out_pages=1), C.ERR_SHAPE), (dict(out_pages=-1), C.ERR_SHAPE),
                      (dict(out_pages=2 ** 60), C.ERR_SHAPE), (dict(w_len=63), C.ERR_SHAPE), (dict(w=None), C.ERR_ARG),
                      (dict(out=None), C.ERR_ARG), (dict(index=None), C.ERR_ARG), (dict(new=None), C.ERR_ARG),
                      (dict(w=FAKE + 1), C.ERR_ALIGN), (dict(kept=FAKE + 2), C.ERR_ALIGN)):
        assert _evict(c, **bad) == code, bad


def test_workspace_of_huge_masks():
    """Sinks and windows past every length change nothing."""
    one = lambda w, s: C.load().lsmx_kv_attend_workspace(ctypes.byref(cache(max_pages=4096)), 1, 4, w, s, 0)  # noqa: E731
    assert one(0, 0) == one(2 ** 63 - 1, 2 ** 63 - 1) == one(5, 2 ** 63 - 1)
    assert one(5, 0) <= one(0, 0)


def test_cpu_tensors_are_refused():
    from lockstep_amd import kv_cache as kc
    from lockstep_amd.attention import sink_window_attention
    q, k = torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gfx950"):
        sink_window_attention(q, k, k)
    with pytest.raises(TypeError):
        sink_window_attention(q.float(), k, k)
    pages = kc.new_pages(4, 2, 64, 16, device="cpu")
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    w = torch.zeros(1, 2, 32)
    for call in (lambda: kc.append(pages, k, k, table, lengths), lambda: kc.attend(q, pages, table, lengths),
                 lambda: kc.evict(pages, table, lengths, w, 2, table)):
        with pytest.raises(RuntimeError, match="gfx950"):
            call()


@pytest.mark.parametrize("src", ["attention.hip", "attention_bwd.hip", "kv_cache.hip"])
def test_kernels_use_no_scratch(src, tmp_path):
    """A spill in a pipelined loop waits for every load in flight."""
    from lockstep_amd import build as B
    flags = [f for f in B.FLAGS if f not in ("-shared", "-fPIC")]
    res = subprocess.run([_hipcc(), *flags, "-c", "-o", str(tmp_path / "k.o"), str(CSRC / src),
                          "-Rpass-analysis=kernel-resource-usage"], capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-2000:]
    scratch = [int(x) for x in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", res.stderr)]
    assert scratch and not any(scratch), f"{src}: {scratch}"

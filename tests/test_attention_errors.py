"""The error of the gradients against 64 bits, as a multiple of what rounding the exact
result to the inputs' type costs.

dQ sums dS_ij k_j with the dS of a row adding up to 0: a common part of the keys
cancels, and with it nearly all of the result's magnitude, but not the roundings
of dS.  With dS rounded once the multiple is 1.4 and more (1.42 where the keys have
no common part, 2.5 with one of twice their spread); with dS in two terms what is left
is the result's own rounding and fp32's.  The limit of 1.25 lies between them.

o, dK and dV have one rounding of each P or dS, and their own, of the same size:
sqrt(2), here at most 1.6."""

import math

import pytest
import torch

CASES = [(700, 64, None, 0, 0.0), (700, 64, None, 0, 2.0), (700, 128, 100, 4, 2.0), (300, 80, None, 0, 4.0)]
DTYPES = [torch.bfloat16, torch.float16]
LIMIT = 1.25


def inputs(T, D, common, dt, heads=2):
    """q, dO [heads, T, D] of one key head, k, v [T, D]."""
    g = torch.Generator().manual_seed(T + D)
    q, do = (torch.randn((heads, T, D), generator=g).to(dt) for _ in range(2))
    k, v = (torch.randn((T, D), generator=g) + common).to(dt), torch.randn((T, D), generator=g).to(dt)
    return q, k, v, do


def formula(q, k, v, do, window, sinks):
    q, k, v, do = (t.double() for t in (q, k, v, do))
    T, D = k.shape
    p, j = torch.arange(T, device=k.device)[:, None], torch.arange(T, device=k.device)
    see = j <= p
    if window:
        see = see & ((j > p - window) | (j < sinks))
    P = torch.softmax(((q @ k.T) / math.sqrt(D)).masked_fill(~see, -math.inf), -1)
    o = P @ v
    dS = P * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(D)
    return {"o": o, "dq": dS @ k, "dk": (dS.transpose(1, 2) @ q).sum(0), "dv": (P.transpose(1, 2) @ do).sum(0), "dS": dS}


def multiple(x, ref, dt):
    return ((x.double() - ref).norm() / (ref.to(dt).double() - ref).norm()).item()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_the_limit_tells_one_term_from_two(case, dt):
    """On the CPU: dQ from dS rounded once, in two terms, and the limit."""
    T, D, window, sinks, common = case
    q, k, v, do = inputs(T, D, common, dt)
    ref = formula(q, k, v, do, window, sinks)
    top = ref["dS"].abs().amax(-1, keepdim=True)   # fp16: into its range, by row
    unit = torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-300))) - 10) if dt == torch.float16 else 1.0
    one = (ref["dS"] / unit).to(dt).double()
    two = one + (ref["dS"] / unit - one).to(dt).double()
    got = [multiple(((x * unit) @ k.double()).to(dt), ref["dq"], dt) for x in (one, two)]
    assert got[0] > LIMIT > got[1]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_errors_of_the_kernels(case, dt, dev):
    from lockstep_amd.attention import sink_window_attention
    T, D, window, sinks, common = case
    q, k, v, do = (t.to(dev) for t in inputs(T, D, common, dt))
    ref = formula(q, k, v, do, window, sinks)
    x = [t[None].contiguous().requires_grad_(True) for t in (q.transpose(0, 1), k[:, None], v[:, None])]
    o = sink_window_attention(*x, window=window, sinks=sinks)
    dq, dk, dv = torch.autograd.grad(o, x, do.transpose(0, 1)[None])
    got = {"dq": multiple(dq[0].transpose(0, 1), ref["dq"], dt), "o": multiple(o[0].detach().transpose(0, 1), ref["o"], dt),
           "dk": multiple(dk[0, :, 0], ref["dk"], dt), "dv": multiple(dv[0, :, 0], ref["dv"], dt)}
    print({n: round(m, 3) for n, m in got.items()}, flush=True)
    assert got["dq"] < LIMIT, got
    assert all(got[n] < 1.6 for n in ("o", "dk", "dv")), got


@pytest.mark.gpu
def test_rows_whose_weight_is_on_the_sinks(dev):
    """A window of one key and four sinks: rows that look at a sink alone take nothing
    from their own key, element by element."""
    from lockstep_amd.attention import sink_window_attention

    from .test_gpu_attention import U, close
    from .test_gpu_attention import formula as bounds
    g = torch.Generator(device=dev).manual_seed(814236)
    x = [torch.randn((2, 560, h, 64), generator=g, device=dev).bfloat16().requires_grad_(True) for h in (9, 3, 3)]
    do = torch.randn((2, 560, 9, 64), generator=g, device=dev).bfloat16()
    dq, = torch.autograd.grad(sink_window_attention(*x, window=1, sinks=4), x[:1], do)
    for b in range(2):
        ref = bounds(*(t[b].detach() for t in x), 1, 4, 0.125, do[b])
        close("dq", dq[b], ref["dq"], ref["dq_mag"], U[torch.bfloat16], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("T,heads", [(64, 1), (64, 48), (200, 2)])
def test_a_nan_key_ahead_does_not_reach_the_rows_behind(T, heads, dev):
    """Key 40 is NaN: the first 32 rows have the dQ that they have without it."""
    from lockstep_amd.attention import sink_window_attention
    for D in (64, 128):
        g = torch.Generator(device=dev).manual_seed(T)
        q, k, v, do = (torch.randn((8, T, heads, D), generator=g, device=dev).bfloat16() for _ in range(4))
        bad = k.clone()
        bad[:, 40] = math.nan
        got = []
        for keys in (k, bad):
            x = [t.clone().requires_grad_(True) for t in (q, keys, v)]
            got.append(torch.autograd.grad(sink_window_attention(*x), x[:1], do)[0])
        assert torch.equal(got[0][:, :32], got[1][:, :32]) and torch.isnan(got[1][:, 40:]).all()

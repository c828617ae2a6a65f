"""fp16 rows over caches whose values fp16 does not hold: written from bf16 with
magnitudes past 65504 or far below fp16's spacing, or exponents set by hand.

Tolerances as in test_gpu_kv_cache.py, with U of fp16, and fp16's spacing near
zero (2^-24, half of it rounding) on the result."""

import math

import pytest
import torch

from .test_gpu_attention import U
from .test_gpu_kv_cache import filled, formula

pytestmark = pytest.mark.gpu


def read(pages, table, b, n, page, Hkv, D, dev):
    """The values that sequence b holds, [n, Hkv, D] in 64 bits."""
    j = torch.arange(n, device=dev)
    pg = table[b, j // page].long()
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=dev)
    grid = torch.cat([grid, -grid])
    out = []
    for c, s in ((0, 1), (2, 3)):
        codes, e = pages[c][pg, :, j % page], pages[s][pg, :, j % page]
        x = grid[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
        out.append(x * torch.exp2(e.double() - 127).repeat_interleave(32, -1))
    return out


def check(lens, T, H, Hkv, D, page, window, sinks, keys, values, dev, qscale=1.0, seed=0):
    """keys, values: (lowest, highest) exponent of a block's scale, and the share of
    blocks that have a random one of them (the others 2^-2)."""
    from lockstep_amd import kv_cache as kc
    pages, table, lengths, _, _ = filled(lens, Hkv, D, page, torch.bfloat16, dev, seed=seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    for t, (lo, hi, share) in ((pages.k_scale, keys), (pages.v_scale, values)):
        e = torch.randint(lo + 127, hi + 128, t.shape, generator=g, device=dev)
        t.copy_(torch.where(torch.rand(t.shape, generator=g, device=dev) < share, e, 125))
    q = (qscale * torch.randn((len(lens), T, H, D), generator=g, device=dev)).half()
    w = torch.zeros((len(lens), Hkv, table.shape[1] * page), device=dev)
    o = kc.attend(q, pages, table, lengths, window=window, sinks=sinks, weights=w)
    assert torch.equal(o, kc.attend(q, pages, table, lengths, window=window, sinks=sinks))
    for b, n in enumerate(lens):
        k, v = read(pages, table, b, n, page, Hkv, D, dev)
        ro, mag, rw, err = formula(q[b], k, v, window, sinks, 1.0 / math.sqrt(D))
        tol = 4 * U[torch.float16] * mag + 2.0 ** -24
        fits = ro.abs() + tol < 65504
        bad = torch.where(fits, (o[b].double() - ro).abs() - tol, 0.0)
        assert bad.max().item() <= 0, (b, bad.max().item())
        assert (o[b][ro.abs() - tol > 65520].abs() == math.inf).all()
        bad = (w[b, :, :n].double() - rw).abs() - err - 2.0 ** -22 * rw
        assert bad.max().item() <= 0, (b, bad.max().item())


# rows of a key head: 1, 4 (a wave's 16), 24 (32), 48, 90, 240 (tiles)
ROWS = [([1], 1, 1, 1, 64, 16), ([700, 33], 1, 8, 2, 128, 64), ([300, 40], 6, 8, 2, 64, 32), ([500], 12, 8, 2, 128, 16),
        ([260, 90], 30, 6, 2, 64, 64), ([400, 260], 60, 8, 2, 128, 32), ([3000], 1, 5, 1, 128, 256)]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 3)])
def test_scales_past_fp16(rows, window, sinks, dev):
    # a few large keys and values among ordinary ones, and all of them large
    check(*rows, window, sinks, (11, 16, 0.02), (13, 17, 0.02), dev, qscale=2.0 ** -14)
    check(*rows, window, sinks, (14, 20, 1.0), (-4, 15, 1.0), dev, qscale=2.0 ** -19)


@pytest.mark.parametrize("rows", ROWS)
def test_scales_below_fp16(rows, dev):
    """Keys of 2^-40 under rows of 2^15, values down to nothing in fp16."""
    check(*rows, None, 0, (-26, -9, 1.0), (-30, -8, 0.3), dev, qscale=2.0 ** 12)


@pytest.mark.parametrize("e", [-24, -23, 13, 14])
def test_both_sides_of_the_switch(e, dev):
    """The last scales whose elements fp16 holds, and the first past them."""
    for rows in ROWS:
        check(*rows, None, 0, (e, e, 1.0), (e, e, 1.0), dev, qscale=2.0 ** min(12, -e))


def test_a_cache_written_from_bf16(dev):
    """One value of 1e5 leaves the rest of its block as it is."""
    from lockstep_amd import kv_cache as kc
    pages = kc.new_pages(2, 1, 64, 16, device=dev)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([1], dtype=torch.int32, device=dev)
    v = torch.full((1, 1, 1, 64), 32768.0, device=dev)
    v[..., 5], v[..., 40] = 1e5, 3.0
    kc.append(pages, torch.zeros_like(v).bfloat16(), v.bfloat16(), table, lengths)
    for T in (1, 40):
        o = kc.attend(torch.zeros((1, T, 2, 64), device=dev).half(), pages, table, lengths)
        assert (o[0, -1, :, 6:32] == 32768).all() and (o[0, -1, :, :5] == 32768).all()
        assert (o[0, -1, :, 5] == math.inf).all()      # 98304 in fp16

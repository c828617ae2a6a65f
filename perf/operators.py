"""The attention operators of this framework, as cases that can be timed.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw()`
others of the same ranges; `prepare()` makes what a program holds before the
call, `run()` is one pass through an operator, `work()` prices it and
`exact()` gives the same outputs in 64 bits.  With `own` set, `run()` calls
the framework; else it computes the operator's plain form from elementary
torch operations in 32 bits, rounded once at the end.

Operators, by "op":
  train    causal attention with a sliding window and sinks, forward and
           gradients (`attention.sink_window_attention`)
  prefill  the same, forward only, over prompts packed one after another
  append   new keys and values written into a paged MXFP4 cache
           (`kv_cache.append`)
  attend   attention of the newest tokens over that cache (`kv_cache.attend`)
  evict    the cache cut down to the tokens with the largest accumulated
           attention weight (`kv_cache.evict`)

The query of token p sees key j when j <= p and (there is no window, or
j > p - window, or j < sinks).  "window": 0 stands for none.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a training step's attention: four query heads share a key head
        {"name": "train_gqa_4096", "op": "train", "dtype": "bf16", "B": 2, "T": 4096, "H": 32, "Hkv": 8, "D": 128,
         "window": 1024, "sinks": 4},
        # a small model's training step at an odd length, every head its own keys
        {"name": "train_f16_777", "op": "train", "dtype": "f16", "B": 3, "T": 777, "H": 12, "Hkv": 12, "D": 64,
         "window": 256, "sinks": 1},
        # eight prompts of different lengths in one prefill, plain causal
        {"name": "prefill_packed", "op": "prefill", "dtype": "bf16", "B": 8, "T": 9000, "H": 16, "Hkv": 4, "D": 128,
         "window": 0, "sinks": 0},
        # one long document through a window with sinks
        {"name": "prefill_long", "op": "prefill", "dtype": "bf16", "B": 1, "T": 16384, "H": 8, "Hkv": 1, "D": 64,
         "window": 4096, "sinks": 16},
        # one new token of each of 64 requests enters the cache
        {"name": "append_decode", "op": "append", "dtype": "bf16", "B": 64, "T": 64, "L": 2048, "Hkv": 8, "D": 128,
         "page": 64},
        # the keys and values of six prompts enter the cache
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "B": 6, "T": 12000, "L": 4096, "Hkv": 8, "D": 128,
         "page": 64},
        # one request, one token, a short cache in small pages: the smallest call
        {"name": "decode_one", "op": "attend", "dtype": "bf16", "B": 1, "T": 1, "L": 1000, "H": 32, "Hkv": 8, "D": 128,
         "page": 16, "window": 0, "sinks": 0, "weights": False},
        # 64 requests of different lengths decode together and accumulate weights
        {"name": "decode_batch", "op": "attend", "dtype": "bf16", "B": 64, "T": 1, "L": 8192, "H": 32, "Hkv": 8,
         "D": 128, "page": 64, "window": 0, "sinks": 0, "weights": True},
        # few requests with very long caches and few key heads
        {"name": "decode_long", "op": "attend", "dtype": "bf16", "B": 4, "T": 1, "L": 100000, "H": 16, "Hkv": 2,
         "D": 128, "page": 256, "window": 0, "sinks": 0, "weights": False},
        # a chunk of a prompt over what is cached of it, windowed, with weights
        {"name": "chunk_600", "op": "attend", "dtype": "f16", "B": 2, "T": 600, "L": 5000, "H": 16, "Hkv": 4, "D": 64,
         "page": 32, "window": 2048, "sinks": 4, "weights": True},
        # one request's cache cut to its budget
        {"name": "evict_one", "op": "evict", "B": 1, "L": 1500, "Hkv": 8, "D": 128, "page": 64, "keep": 1024,
         "sinks": 4, "recent": 128},
        # a batch's caches halved
        {"name": "evict_batch", "op": "evict", "B": 32, "L": 8192, "Hkv": 8, "D": 128, "page": 64, "keep": 4096,
         "sinks": 4, "recent": 512},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice((1, 2, 3, 4, 8))
    return hkv * rng.choice((1, 2, 4, 5, 8)), hkv


def draw(rng):
    op = rng.choice(("train", "train", "prefill", "append", "attend", "attend", "attend", "evict"))
    while True:
        c = {"op": op}
        if op != "evict":
            c["dtype"] = rng.choice(("bf16", "bf16", "f16"))
        if op in ("train", "prefill"):
            h, hkv = _heads(rng)
            c.update(B=rng.choice((1, 2, 3, 5, 8)), T=_log(rng, 64, 16384), H=h, Hkv=hkv, D=rng.choice((64, 80, 96, 128)),
                     window=rng.choice((0, _log(rng, 16, 4096))), sinks=rng.choice((0, 1, 4, 16, 100)))
            if op == "prefill" and c["T"] < 8 * c["B"]:
                continue
            pairs = (c["B"] if op == "train" else 1) * h * c["T"] ** 2
            ok = pairs <= (1.0e9 if op == "train" else 2.1e9)
        elif op == "append":
            c.update(B=rng.choice((1, 3, 6, 32, 64)), Hkv=rng.choice((1, 2, 4, 8)), D=rng.choice((64, 128)),
                     page=rng.choice((16, 32, 64, 128, 256)), L=_log(rng, 64, 4096))
            c["T"] = c["B"] if rng.random() < 0.4 else _log(rng, c["B"], 12000)
            ok = c["T"] <= c["B"] * c["L"] // 2
        elif op == "attend":
            h, hkv = _heads(rng)
            c.update(B=_log(rng, 1, 64), L=_log(rng, 64, 100000), H=h, Hkv=hkv, D=rng.choice((64, 128)),
                     T=rng.choice((1, 1, 1, 2, 5, _log(rng, 8, 600))), page=rng.choice((16, 32, 64, 128, 256)),
                     window=rng.choice((0, 0, _log(rng, 64, 8192))), sinks=rng.choice((0, 4, 16)),
                     weights=rng.random() < 0.4)
            ok = c["T"] <= c["L"] and c["B"] * hkv * c["L"] <= 4.2e6 and c["B"] * h * c["T"] * c["L"] <= 1.0e8
        else:
            c.update(B=rng.choice((1, 2, 7, 16, 32)), L=_log(rng, 128, 16384), Hkv=rng.choice((1, 2, 4, 8)),
                     D=rng.choice((64, 128)), page=rng.choice((16, 32, 64, 128, 256)), sinks=rng.choice((0, 4, 16)))
            c["keep"] = max(32, int(c["L"] * rng.uniform(0.2, 0.9)))
            c["recent"] = int((c["keep"] - c["sinks"]) * rng.uniform(0.0, 0.5))
            ok = c["B"] * c["Hkv"] * c["L"] <= 2.1e6
        if ok:
            return c


# ------------------------------------------------------------------ raggedness
def _split(total, n):
    """`total` tokens in n sequences of different lengths, one at least each."""
    w = [1 + (5 * i + 2) % 7 for i in range(n)]
    got = [max(1, total * x // sum(w)) for x in w]
    got[0] += total - sum(got)
    return got


def _lengths(c):
    """Tokens in the cache of each request: L for the first, down to half of it."""
    return [max(c.get("T", 1) if c["op"] == "attend" else 1, c["L"] - c["L"] * ((37 * b) % 64) // 128)
            for b in range(c["B"])]


def _new_tokens(c):
    """New tokens of each request in an append, and its length with them."""
    new = _split(c["T"], c["B"])
    return new, [max(n, c["L"] - (29 * b) % (c["L"] // 2 + 1)) for b, n in enumerate(new)]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dt):
    return torch.randn(shape, generator=g, device="cuda").to(dt)


def _keys(g, shape, dt):
    """Keys: normal, with channels of different size."""
    s = torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda") * s).to(dt)


def _inputs(c, seed):
    """The plain tensors that both prepare() and exact() start from, cached
    tokens in their order."""
    g, op, D = _gen(seed), c["op"], c["D"]
    dt = _DT[c.get("dtype", "bf16")]
    if op == "train":
        q, o = (c["B"], c["T"], c["H"], D), (c["B"], c["T"], c["Hkv"], D)
        return {"q": _normal(g, q, dt), "k": _keys(g, o, dt), "v": _normal(g, o, dt), "do": _normal(g, q, dt)}
    if op == "prefill":
        o = (c["T"], c["Hkv"], D)
        return {"q": _normal(g, (c["T"], c["H"], D), dt), "k": _keys(g, o, dt), "v": _normal(g, o, dt)}
    if op == "append":
        o = (c["T"], c["Hkv"], D)
        return {"k": _keys(g, o, dt), "v": _normal(g, o, dt)}
    o = (c["B"], max(_lengths(c)), c["Hkv"], D)
    t = {"k": _keys(g, o, dt), "v": _normal(g, o, dt)}
    if op == "attend":
        t["q"] = _normal(g, (c["B"], c["T"], c["H"], D), dt)
    if op == "evict" or c["weights"]:
        # accumulated weights: long tailed, some tokens never looked at
        w = torch.exp(2.0 * torch.randn((c["B"], c["Hkv"], o[1]), generator=g, device="cuda"))
        t["weights"] = torch.where(w < 0.2, torch.zeros_like(w), w)
    return t


def _tables(counts, seed, first=0):
    """A block table: `counts` pages for each request, scattered over the
    pool from page `first` on, -1 past a request's last."""
    n = sum(counts)
    perm = (torch.randperm(n, generator=torch.Generator().manual_seed(seed)) + first).to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32)
    at = torch.arange(max(counts))[None] < torch.tensor(counts)[:, None]
    table[at] = perm
    return table.cuda(), n


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(pages, c):
    D = c["D"]
    one = lambda n: torch.zeros((pages, c["Hkv"], c["page"], n), dtype=torch.uint8, device="cuda")  # noqa: E731
    return [one(D // 2), one(D // 32), one(D // 2), one(D // 32)]


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    op = c["op"]
    t["case"] = c
    if op == "train":
        for n in ("q", "k", "v"):
            t[n].requires_grad_(True)
        return t
    if op == "prefill":
        lens = _split(c["T"], c["B"])
        t["offsets"] = _int32([sum(lens[:b]) for b in range(c["B"] + 1)])
        return t
    if op == "append":
        new, lens = _new_tokens(c)
        t["offsets"] = _int32([sum(new[:b]) for b in range(c["B"] + 1)])
    else:
        lens = _lengths(c)
    t["lengths"] = _int32(lens)
    t["table"], n = _tables([-(-x // c["page"]) for x in lens], seed)
    if op == "append":
        t["pages"] = _pool(n, c)
        return t
    more = 0
    if op == "evict":
        t["out_table"], more = _tables([-(-min(x, c["keep"]) // c["page"]) for x in lens], seed + 1, n)
        t["out_first"] = n
    if "weights" in t:  # as wide as the table
        w = torch.zeros((c["B"], c["Hkv"], t["table"].shape[1] * c["page"]), device="cuda")
        w[:, :, :t["weights"].shape[2]] = t["weights"]
        t["weights"] = w
    t["pages"] = _pool(n + more, c)
    b, j = torch.nonzero(torch.arange(max(lens), device="cuda")[None] < t["lengths"][:, None], as_tuple=True)
    _store(t["pages"], t.pop("k")[b, j], t.pop("v")[b, j], t["table"][b, j // c["page"]].long(), j % c["page"])
    return t


# ------------------------------------------------------------------ plain forms
def _quantize(x):
    """x [..., D] in MXFP4 blocks of 32: codes (0..15) [..., D], biased
    exponents [..., D / 32], and the values they stand for."""
    b = x.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.where(amax == 0, 0, torch.frexp(amax).exponent - 3)  # floor(log2) - 2
    e = e.clamp(min=-102)
    s = ((e + 127).to(torch.int32) << 23).view(torch.float32)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    mag = torch.bucketize(b.abs() / s, mids)
    codes = mag + 8 * torch.signbit(b)
    return codes.flatten(-2).to(torch.uint8), (e + 127).squeeze(-1).to(torch.uint8), (_e2m1(codes) * s).flatten(-2)


def _e2m1(codes):
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    return torch.cat([v, -v])[codes.long()]


def _store(pages, k, v, page, at):
    """k, v [n, Hkv, D] into slots `at` of pages `page`; their values back."""
    kc, ke, kv = _quantize(k)
    vc, ve, vv = _quantize(v)
    pages[0][page, :, at] = kc[..., ::2] | kc[..., 1::2] << 4
    pages[1][page, :, at] = ke
    pages[2][page, :, at] = vc[..., ::2] | vc[..., 1::2] << 4
    pages[3][page, :, at] = ve
    return kv, vv


def _load(codes, scale, table, page):
    """The cached tokens of every request, [B, Hkv, tokens, D] in 32 bits."""
    at = table.clamp(min=0).long()
    c, e = codes[at].transpose(1, 2).flatten(2, 3), scale[at].transpose(1, 2).flatten(2, 3)
    v = _e2m1(torch.stack([c & 15, c >> 4], -1).flatten(-2))
    return v * (e.to(torch.int32) << 23).view(torch.float32).repeat_interleave(32, -1)


def _fold(q, hkv):
    """[B, T, H, D] -> [B, Hkv, group * T, D] in 32 bits."""
    return q.float().unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)


def _unfold(o, T):
    return o.unflatten(2, (-1, T)).permute(0, 3, 1, 2, 4).flatten(2, 3)


def _sees(p, j, window, sinks):
    return (j <= p) & ((j > p - window) | (j < sinks) if window else j <= p)


def _softmax(q, k, mask, group):
    """Probabilities [B, Hkv, group * T, keys]; rows that see nothing are 0."""
    s = q @ k.transpose(-1, -2) * (1.0 / math.sqrt(q.shape[-1]))
    s = torch.where(mask.repeat(1, 1, group, 1), s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _plain_train(t, c):
    T, hkv, dt, j = c["T"], c["Hkv"], t["q"].dtype, torch.arange(c["T"], device="cuda")
    q, do = _fold(t["q"], hkv), _fold(t["do"], hkv)
    k, v = t["k"].float().transpose(1, 2), t["v"].float().transpose(1, 2)
    p = _softmax(q, k, _sees(j[:, None], j, c["window"], c["sinks"])[None, None], c["H"] // hkv)
    o = p @ v
    ds = do @ v.transpose(-1, -2)
    ds = p * (ds - (do * o).sum(-1, keepdim=True)) * (1.0 / math.sqrt(c["D"]))
    dk, dv = ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ do
    return {"o": _unfold(o, T).to(dt), "dq": _unfold(ds @ k, T).to(dt), "dk": dk.transpose(1, 2).to(dt),
            "dv": dv.transpose(1, 2).to(dt)}


def _plain_prefill(t, c):
    i = torch.arange(c["T"], device="cuda")
    seq = torch.searchsorted(t["offsets"], i.to(torch.int32), right=True) - 1
    at = i - t["offsets"][seq]
    mask = _sees(at[:, None], at, c["window"], c["sinks"]) & (seq[:, None] == seq)
    k, v = t["k"].float().transpose(0, 1)[None], t["v"].float().transpose(0, 1)[None]
    p = _softmax(_fold(t["q"][None], c["Hkv"]), k, mask[None, None], c["H"] // c["Hkv"])
    return _unfold(p @ v, c["T"])[0].to(t["q"].dtype)


def _plain_append(t, c):
    i = torch.arange(c["T"], device="cuda")
    seq = torch.searchsorted(t["offsets"], i.to(torch.int32), right=True) - 1
    j = t["lengths"][seq] - (t["offsets"][seq + 1] - i)
    k, v = _store(t["pages"], t["k"], t["v"], t["table"][seq, j // c["page"]].long(), j % c["page"])
    return {"k": k.bfloat16(), "v": v.bfloat16()}


def _plain_attend(t, c):
    pages, n = t["pages"], t["lengths"].long()
    j = torch.arange(t["table"].shape[1] * c["page"], device="cuda")
    k, v = _load(pages[0], pages[1], t["table"], c["page"]), _load(pages[2], pages[3], t["table"], c["page"])
    at = n[:, None, None] - c["T"] + torch.arange(c["T"], device="cuda")[:, None]
    p = _softmax(_fold(t["q"], c["Hkv"]), k, _sees(at, j, c["window"], c["sinks"])[:, None], c["H"] // c["Hkv"])
    o = _unfold(p @ v, c["T"]).to(t["q"].dtype)
    if not c["weights"]:
        return o
    t["weights"].add_(p.sum(2))
    return {"o": o, "weights": t["weights"]}


def _plain_evict(t, c):
    n, w, keep = t["lengths"][:, None, None], t["weights"], c["keep"]
    j = torch.arange(w.shape[2], device="cuda")
    rank = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), math.inf, w)
    rank = torch.where(j < n, rank, -1.0)
    index = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    index = torch.sort(torch.where(index < n, index, w.shape[2]), dim=2).values
    index = torch.nn.functional.pad(index, (0, keep - index.shape[2]), value=w.shape[2])
    held = index < n
    b, h, to = torch.nonzero(held, as_tuple=True)
    src, page = index[b, h, to], c["page"]
    fp, tp = t["table"][b, src // page].long(), t["out_table"][b, to // page].long()
    pages = t["pages"]
    pages[0][tp, h, to % page], pages[1][tp, h, to % page] = pages[0][fp, h, src % page], pages[1][fp, h, src % page]
    pages[2][tp, h, to % page], pages[3][tp, h, to % page] = pages[2][fp, h, src % page], pages[3][fp, h, src % page]
    kept = torch.where(held, w.gather(2, index.clamp(max=w.shape[2] - 1)), 0.0)
    return torch.where(held, index, -1).to(torch.int32), kept, t["lengths"].clamp(max=keep)


# ------------------------------------------------------------------ one pass
def run(t):
    c = t["case"]
    if not own:
        with torch.no_grad():
            got = globals()["_plain_" + c["op"]](t, c)
        return _with_moved(t, got) if c["op"] == "evict" else got
    if c["op"] in ("train", "prefill"):
        from lockstep_amd.attention import sink_window_attention

        window = c["window"] or None
        if c["op"] == "prefill":
            return sink_window_attention(t["q"], t["k"], t["v"], window=window, sinks=c["sinks"],
                                         offsets=t["offsets"])
        o = sink_window_attention(t["q"], t["k"], t["v"], window=window, sinks=c["sinks"])
        dq, dk, dv = torch.autograd.grad(o, (t["q"], t["k"], t["v"]), t["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    from lockstep_amd import kv_cache

    pages = kv_cache.Pages(*t["pages"])
    if c["op"] == "append":
        k, v = kv_cache.append(pages, t["k"], t["v"], t["table"], t["lengths"], offsets=t["offsets"], values=True)
        return {"k": k, "v": v}
    if c["op"] == "attend":
        o = kv_cache.attend(t["q"], pages, t["table"], t["lengths"], window=c["window"] or None, sinks=c["sinks"],
                            weights=t.get("weights"))
        return {"o": o, "weights": t["weights"]} if c["weights"] else o
    got = kv_cache.evict(pages, t["table"], t["lengths"], t["weights"], c["keep"], t["out_table"], sinks=c["sinks"],
                         recent=c["recent"])
    return _with_moved(t, got)


def _with_moved(t, got):
    """An eviction's answers and the pages it filled.  Their bytes (two codes
    each, or a block's exponent) are moved, not computed: they come as they
    are held."""
    index, weights, lengths = got
    kc, ke, vc, ve = (x[t["out_first"]:] for x in t["pages"])
    return {"index": index, "weights": weights, "lengths": lengths, "kc": kc, "ke": ke, "vc": vc, "ve": ve}


# ------------------------------------------------------------------ its price
def _pairs(queries, keys, window, sinks):
    """Visible (query, key) pairs of the last `queries` tokens of `keys`."""
    near = lambda p: min(p + 1, window) if window else p + 1  # noqa: E731
    return sum(near(p) + min(sinks, p + 1 - near(p)) for p in range(keys - queries, keys))


def work(case):
    """Bytes read and written once, and multiply-adds times two."""
    c, op, D = case, case["op"], case["D"]
    held = D // 2 + D // 32  # bytes of one head's vector of one token in MXFP4
    if op == "train":
        n = c["B"] * c["T"]
        pairs = c["B"] * _pairs(c["T"], c["T"], c["window"], c["sinks"])
        # q, do in, o, dq out; k, v in, dk, dv out; two products forward, five backward
        return {"bytes": 2.0 * n * D * 4 * (c["H"] + c["Hkv"]), "flops": 14.0 * D * c["H"] * pairs}
    if op == "prefill":
        pairs = sum(_pairs(n, n, c["window"], c["sinks"]) for n in _split(c["T"], c["B"]))
        return {"bytes": 2.0 * c["T"] * D * 2 * (c["H"] + c["Hkv"]), "flops": 4.0 * D * c["H"] * pairs}
    if op == "append":  # both in, their codes and scales and their values out
        return {"bytes": 2.0 * c["T"] * c["Hkv"] * (2 * D + held + 2 * D), "flops": 0.0}
    lens = _lengths(c)
    if op == "attend":
        seen = [n if not c["window"] else min(n, c["window"] + c["T"] - 1 + c["sinks"]) for n in lens]
        moved = c["Hkv"] * sum(seen) * (2 * held + (8 if c["weights"] else 0)) + 4.0 * c["B"] * c["T"] * c["H"] * D
        pairs = sum(_pairs(c["T"], n, c["window"], c["sinks"]) for n in lens)
        return {"bytes": moved, "flops": 4.0 * D * c["H"] * pairs}
    kept = sum(min(n, c["keep"]) for n in lens)
    return {"bytes": c["Hkv"] * (4.0 * sum(lens) + kept * (4 * held + 8)), "flops": 0.0}


# ------------------------------------------------------------------ in 64 bits
def _values64(x):
    """The values MXFP4 holds for x [..., D], in float64: blocks of 32 along
    D, scale 2^(floor(log2(amax)) - 2), elements to the nearest of the grid,
    ties to the smaller."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-30))) - 2))
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device, dtype=torch.float64)
    r = (b.abs() / scale).clamp(max=6.0)
    up = torch.searchsorted(grid, r).clamp(min=1)
    lo, hi = grid[up - 1], grid[up]
    return (torch.where(r - lo <= hi - r, lo, hi) * torch.sign(b) * scale).flatten(-2)


def _attention64(q, k, v, first, window, sinks, do=None):
    """One key head: q [T, G, D] of the tokens from `first` on, k, v [n, D]."""
    n, D = k.shape
    p0 = first + torch.arange(q.shape[0], device="cuda")
    j = torch.arange(n, device="cuda")
    hide = j[None] > p0[:, None]
    if window:
        hide |= (j[None] <= p0[:, None] - window) & (j[None] >= sinks)
    o, dq, dk, dv, w = [], [], torch.zeros_like(k), torch.zeros_like(v), torch.zeros(n, device="cuda", dtype=k.dtype)
    for h in range(q.shape[1]):
        s = (q[:, h] @ k.t() / math.sqrt(D)).masked_fill_(hide, -math.inf)
        p = torch.softmax(s, -1)
        w += p.sum(0)
        o.append(p @ v)
        if do is not None:
            g = p * (do[:, h] @ v.t() - (do[:, h] * o[-1]).sum(-1, keepdim=True)) / math.sqrt(D)
            dq.append(g @ k)
            dk += g.t() @ q[:, h]
            dv += p.t() @ do[:, h]
    return torch.stack(o, 1), w, torch.stack(dq, 1) if dq else None, dk, dv


def exact(case, seed):
    c, op, t = case, case["op"], _inputs(case, seed)
    G = c.get("H", 1) // c["Hkv"]
    if op == "append":
        return {"k": _values64(t["k"]), "v": _values64(t["v"])}
    if op == "evict":
        kept = torch.zeros((c["B"], c["Hkv"], c["keep"]), device="cuda", dtype=torch.float64)
        for b, n in enumerate(_lengths(c)):
            for h in range(c["Hkv"]):
                w = t["weights"][b, h, :n].cpu().tolist()
                free = range(min(c["sinks"], n), max(min(c["sinks"], n), n - c["recent"]))
                best = sorted(free, key=lambda x: (-w[x], x))[:max(0, c["keep"] - (n - len(free)))]
                took = sorted([x for x in range(n) if x not in free] + best)
                kept[b, h, :len(took)] = torch.tensor([w[x] for x in took], dtype=torch.float64)
        return {"index": None, "weights": kept, "lengths": None, "kc": None, "ke": None, "vc": None, "ve": None}
    if op == "prefill":
        out, at = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64), 0
        for n in _split(c["T"], c["B"]):
            for h in range(c["Hkv"]):
                q, k, v = t["q"][at:at + n, h * G:(h + 1) * G], t["k"][at:at + n, h], t["v"][at:at + n, h]
                out[at:at + n, h * G:(h + 1) * G] = _attention64(q.double(), k.double(), v.double(), 0, c["window"],
                                                                 c["sinks"])[0]
            at += n
        return out
    o = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)
    if op == "attend":
        wide = -(-max(_lengths(c)) // c["page"]) * c["page"]
        w = torch.zeros((c["B"], c["Hkv"], wide), device="cuda", dtype=torch.float64)
        if c["weights"]:
            w[:, :, :t["weights"].shape[2]] = t["weights"]
        for b, n in enumerate(_lengths(c)):
            k, v = _values64(t["k"][b, :n]), _values64(t["v"][b, :n])
            for h in range(c["Hkv"]):
                got = _attention64(t["q"][b, :, h * G:(h + 1) * G].double(), k[:, h], v[:, h], n - c["T"], c["window"],
                                   c["sinks"])
                o[b, :, h * G:(h + 1) * G] = got[0]
                w[b, h, :n] += got[1]
        return {"o": o, "weights": w} if c["weights"] else o
    dq = torch.zeros_like(o)
    dk = torch.zeros(t["k"].shape, device="cuda", dtype=torch.float64)
    dv = torch.zeros_like(dk)
    for b in range(c["B"]):
        for h in range(c["Hkv"]):
            at = slice(h * G, (h + 1) * G)
            q, k, v, do = t["q"][b, :, at], t["k"][b, :, h], t["v"][b, :, h], t["do"][b, :, at]
            got = _attention64(q.double(), k.double(), v.double(), 0, c["window"], c["sinks"], do.double())
            o[b, :, at], dq[b, :, at], dk[b, :, h], dv[b, :, h] = got[0], got[2], got[3], got[4]
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}

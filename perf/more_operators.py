"""The norm, the router and the experts' products, as cases that can be timed.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw()`
others of the same ranges; `prepare()` makes what a program holds before the
call, `run()` is one pass through an operator, `work()` prices it and
`exact()` gives the same outputs in 64 bits.  With `own` set, `run()` calls
the framework; else it computes the operator's plain form from elementary
torch operations in 32 bits, rounded once at the end.

Operators, by "op":
  norm     the residual added, a root-mean-square norm, and its output in
           MXFP8 beside the plain one (`norm.add_rms_norm`)
  train    the same without MXFP8, forward and gradients
  route    a router's choice of experts and their weights; with "grad" the
           gradient of the logits too (`experts.route`)
  gated    the (token, expert) pairs sorted by expert and the experts' first
           product: gate and up rows, silu(gate) * up, in MXFP8
           (`experts.dispatch`, `experts.expert_gated`)
  combine  the experts' second product, summed over each token's experts with
           their weights (`experts.expert_combine`)

MXFP8: E4M3 codes with one power-of-two scale for 32 along the row, the least
that keeps the block within 448.  MXFP4: two E2M1 codes a byte, scales alike.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # eight requests' next tokens between two layers: the smallest call
        {"name": "norm_decode", "op": "norm", "dtype": "bf16", "T": 8, "D": 4096},
        # a prompt's tokens between two layers
        {"name": "norm_prompt", "op": "norm", "dtype": "bf16", "T": 8192, "D": 8192},
        # a training step at an odd number of tokens
        {"name": "norm_train", "op": "train", "dtype": "f16", "T": 8190, "D": 4096},
        # one decoding step of 64 requests, experts in groups, balanced by a bias
        {"name": "route_decode", "op": "route", "dtype": "f32", "T": 64, "E": 256, "k": 8, "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renorm": True, "grad": False},
        # a training step's router
        {"name": "route_train", "op": "route", "dtype": "bf16", "T": 16384, "E": 64, "k": 6, "scoring": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "renorm": True, "grad": True},
        # prompts through a router of many experts
        {"name": "route_prompt", "op": "route", "dtype": "f32", "T": 30001, "E": 256, "k": 8, "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renorm": True, "grad": False},
        # one request decodes: its four experts are read, little else
        {"name": "gated_one", "op": "gated", "T": 1, "K": 2048, "F": 1024, "E": 32, "k": 4, "padded": 0},
        # 64 requests decode: nearly every expert is read, for a few rows each
        {"name": "gated_decode", "op": "gated", "T": 64, "K": 4096, "F": 1024, "E": 128, "k": 8, "padded": 0},
        # prompts, packed into a batch with padding behind them
        {"name": "gated_prompt", "op": "gated", "T": 8192, "K": 4096, "F": 2048, "E": 32, "k": 4, "padded": 500},
        # five requests decode
        {"name": "combine_few", "op": "combine", "dtype": "bf16", "T": 5, "K": 1024, "N": 2048, "E": 32, "k": 4,
         "padded": 0},
        # a chunk of a prompt, a few dozen rows for each expert
        {"name": "combine_chunk", "op": "combine", "dtype": "f16", "T": 333, "K": 1408, "N": 2048, "E": 64, "k": 6,
         "padded": 13},
        # prompts: the second product of gated_prompt
        {"name": "combine_prompt", "op": "combine", "dtype": "bf16", "T": 8192, "K": 2048, "N": 4096, "E": 32, "k": 4,
         "padded": 500},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "train", "route", "route", "gated", "gated", "combine", "combine"))
    while True:
        c = {"op": op}
        if op in ("norm", "train"):
            c.update(dtype=rng.choice(("bf16", "bf16", "f16", "f32")), T=_log(rng, 1, 16384))
            c["D"] = 32 * _log(rng, 8, 256) if op == "norm" or rng.random() < 0.6 else _log(rng, 200, 8200)
            ok = c["T"] * c["D"] <= (2 ** 26 if op == "norm" else 2 ** 25)
        elif op == "route":
            groups = rng.choice((1, 1, 4, 8))
            c.update(dtype=rng.choice(("f32", "f32", "bf16", "f16")), T=_log(rng, 1, 30000),
                     E=groups * rng.choice((4, 8, 15, 16, 32, 48)), scoring=rng.choice(("softmax", "sigmoid")),
                     bias=rng.random() < 0.5, groups=groups, top_groups=max(1, groups // 2), renorm=rng.random() < 0.7,
                     grad=rng.random() < 0.4)
            c["k"] = rng.choice((1, 2, 3, 4, 6, 8))
            ok = c["k"] <= c["E"] // groups * c["top_groups"] and c["T"] * c["E"] <= 7.6e6
        else:
            c.update(T=_log(rng, 1, 8192), K=128 * _log(rng, 4, 32), E=rng.choice((4, 8, 16, 32, 60, 64, 128)),
                     k=rng.choice((1, 2, 4, 6, 8)))
            c["padded"] = rng.choice((0, 0, c["T"] // 7))
            if op == "gated":
                c["F"] = 32 * _log(rng, 8, 64)
                cost = 2 * c["F"] * c["K"]
            else:
                c["N"] = 32 * _log(rng, 16, 128)
                c["dtype"] = rng.choice(("bf16", "bf16", "f16"))
                cost = c["N"] * c["K"]
            ok = (c["k"] <= c["E"] and c["E"] * cost <= 1.0e9 and
                  c["T"] * c["k"] * cost <= (5.4e11 if op == "gated" else 2.7e11))
        if ok:
            return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _packed(g, experts, rows, K):
    """MXFP4 weights of `experts` experts: any codes, scales that keep the
    products near 1."""
    codes = torch.randint(0, 256, (experts, rows, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    mid = 127 - round(math.log2(2.9 * math.sqrt(K)))
    scale = torch.randint(mid - 1, mid + 2, (experts, rows, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    return codes, scale


def _chosen(g, c):
    """Experts of every token, some of them more popular; -1 for the padding
    behind the last token."""
    liking = _randn(g, c["E"]) * 0.5 + _randn(g, c["T"], c["E"])
    ids = liking.topk(c["k"], dim=1).indices.to(torch.int32)
    if c["padded"]:
        ids[c["T"] - c["padded"]:] = -1
    return ids


def _inputs(c, seed):
    g, op, T = _gen(seed), c["op"], c["T"]
    if op in ("norm", "train"):
        dt, D = _DT[c["dtype"]], c["D"]
        wide = torch.exp(0.7 * _randn(g, D))  # channels of different size
        t = {"x": _randn(g, T, D).to(dt), "r": (_randn(g, T, D) * wide).to(dt), "w": (1 + 0.2 * _randn(g, D)).to(dt)}
        if op == "train":
            t["dy"], t["dh"] = _randn(g, T, D).to(dt), _randn(g, T, D).to(dt)
        return t
    if op == "route":
        t = {"logits": (1.5 * _randn(g, T, c["E"]) + 0.5 * _randn(g, c["E"])).to(_DT[c["dtype"]])}
        t["bias"] = 0.1 * _randn(g, c["E"]) if c["bias"] else None
        if c["grad"]:
            t["dw"] = _randn(g, T, c["k"])
        return t
    t = {"experts": _chosen(g, c)}
    rows = T if op == "gated" else T * c["k"]
    t["x"], t["xs"] = _mxfp8(_randn(g, rows, c["K"]) * torch.exp(0.5 * _randn(g, c["K"])))
    t["w"], t["ws"] = _packed(g, c["E"], 2 * c["F"] if op == "gated" else c["N"], c["K"])
    if op == "combine":
        t["x"], t["xs"] = t["x"].view(T, c["k"], -1), t["xs"].view(T, c["k"], -1)
        t["weights"] = torch.softmax(_randn(g, T, c["k"]), 1)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    t["case"] = case
    if case["op"] == "train":
        for n in ("x", "r", "w"):
            t[n].requires_grad_(True)
    if case["op"] == "route" and case["grad"]:
        t["logits"].requires_grad_(True)
    if case["op"] in ("gated", "combine"):
        # the rows of the expert with the most: the plain form's batches are as high
        ids = t["experts"].flatten()
        t["most"] = max(1, int(torch.bincount(ids[ids >= 0].long(), minlength=1).max())) if ids.numel() else 1
        t["order"], t["offsets"] = _sorted(t["experts"], case["E"])
    return t


# ------------------------------------------------------------------ plain forms
def _mxfp8(x):
    """x [.., D] in 32 bits as E4M3 codes and E8M0 bytes."""
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(m == 0, 0, e - 9 + (m > 0.875)).clamp(min=-127)
    codes = torch.ldexp(b, -e[..., None]).flatten(-2)
    return codes.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _power(e):
    """2^(e - 127) of E8M0 bytes, in 32 bits."""
    return torch.ldexp(torch.ones((), device=e.device), e.to(torch.int32) - 127)


def _values8(codes, scale):
    return (codes.float().unflatten(-1, (-1, 32)) * _power(scale)[..., None]).flatten(-2)


def _values4(codes, scale):
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    pairs = torch.cartesian_prod(torch.cat([v, -v]), torch.cat([v, -v])).flip(1)  # of a byte: low nibble first
    return (pairs[codes.int()].unflatten(-2, (-1, 16)).flatten(-2) * _power(scale)[..., None]).flatten(-2)


def _plain_norm(t, c):
    h = (t["x"].float() + t["r"].float()).to(t["x"].dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * t["w"].float()
    codes, scale = _mxfp8(y)
    return {"y": y.to(h.dtype), "h": h, "codes": codes, "scale": scale.view(torch.float8_e8m0fnu)}


def _plain_train(t, c):
    dt = t["x"].dtype
    h = (t["x"].float() + t["r"].float()).to(dt)
    f, w, dy = h.float(), t["w"].float(), t["dy"].float()
    inv = torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)
    n = f * inv
    g = dy * w
    dx = inv * (g - n * (g * n).mean(-1, keepdim=True)) + t["dh"].float()
    return {"y": (n * w).to(dt), "h": h, "dx": dx.to(dt), "dr": dx.to(dt), "dw": (dy * n).sum(0).to(dt)}


def _first(values, k):
    """Indices of the k largest, ties to the lowest index."""
    return torch.sort(values, dim=-1, descending=True, stable=True).indices[..., :k]


def _plain_route(t, c):
    # 64 bits: two experts' scores may lie nearer than 32 bits tell apart
    x = t["logits"].double()
    s = torch.exp(x - x.amax(-1, keepdim=True)) if c["scoring"] == "softmax" else 1.0 / (1.0 + torch.exp(-x))
    if c["scoring"] == "softmax":
        s = s / s.sum(-1, keepdim=True)
    rank = s if t["bias"] is None else s + t["bias"].double()
    if c["groups"] > 1:
        by = rank.unflatten(-1, (c["groups"], -1))
        best = _first(by, 2)
        top = _first(by.gather(-1, best).sum(-1), c["top_groups"])
        keep = torch.zeros(by.shape[:2], dtype=torch.bool, device=x.device).scatter(1, top, True)
        rank = torch.where(keep[..., None], by, -math.inf).flatten(-2)
    at = _first(rank, c["k"])
    a = s.gather(-1, at)
    total = a.sum(-1, keepdim=True) if c["renorm"] else torch.ones_like(a[:, :1])
    got = {"weights": (a / total).float(), "experts": at.to(torch.int32)}
    if c["grad"]:
        dw = t["dw"].double()
        da = (dw - (dw * a).sum(-1, keepdim=True) / total) / total if c["renorm"] else dw
        g = torch.zeros_like(s).scatter(-1, at, da)
        if c["scoring"] == "softmax":
            d = s * (g - (da * a).sum(-1, keepdim=True))
        else:
            d = g * s * (1.0 - s)
        got["dlogits"] = d.to(t["logits"].dtype)
    return got


def _sorted(experts, E):
    """Pairs in the order of their experts (those of none behind), and where
    each expert's begin."""
    ids = experts.flatten()
    ids = torch.where((ids >= 0) & (ids < E), ids, E)
    ids, order = torch.sort(ids, stable=True)
    offsets = torch.searchsorted(ids, torch.arange(E + 1, device=ids.device, dtype=torch.int32))
    return order.to(torch.int32), offsets.to(torch.int32)


def _products(rows, w, ws, experts, order, offsets, most):
    """rows [pairs, K] times their experts' weights, [pairs, N]; 0 for pairs of
    no expert.  One batched product over the experts, each padded to `most`."""
    E, K = w.shape[0], rows.shape[1]
    ids = experts.flatten().long()
    place = torch.empty_like(ids).scatter(0, order.long(), torch.arange(ids.numel(), device=ids.device))
    there = ids >= 0
    at = torch.where(there, ids * most + place - offsets[ids.clamp(min=0)], E * most)
    batch = torch.zeros((E * most + 1, K), device=rows.device).index_copy(0, at, rows)
    wt = _values4(w, ws).transpose(1, 2).contiguous()
    out = torch.bmm(batch[:-1].view(E, most, K), wt).flatten(0, 1)
    return torch.where(there[:, None], out[at.clamp(max=E * most - 1)], 0.0)


def _plain_gated(t, c):
    order, offsets = _sorted(t["experts"], c["E"])
    rows = _values8(t["x"], t["xs"]).repeat_interleave(c["k"], 0)
    gate, up = _products(rows, t["w"], t["ws"], t["experts"], order, offsets, t["most"]).chunk(2, -1)
    h, hs = _mxfp8(gate / (1.0 + torch.exp(-gate)) * up)
    shape = (c["T"], c["k"], -1)
    return {"h": h.view(shape), "scale": hs.view(torch.float8_e8m0fnu).view(shape), "order": order, "offsets": offsets}


def _plain_combine(t, c):
    rows = _values8(t["x"], t["xs"]).flatten(0, 1)
    z = _products(rows, t["w"], t["ws"], t["experts"], t["order"], t["offsets"], t["most"])
    return (z.view(c["T"], c["k"], -1) * t["weights"][..., None]).sum(1).to(_DT[c["dtype"]])


# ------------------------------------------------------------------ one pass
def run(t):
    c = t["case"]
    if not own:
        with torch.no_grad():
            return globals()["_plain_" + c["op"]](t, c)
    if c["op"] in ("norm", "train"):
        from lockstep_amd.norm import add_rms_norm

        if c["op"] == "norm":
            y, h, codes, scale = add_rms_norm(t["x"], t["w"], t["r"], mxfp8=True)
            return {"y": y, "h": h, "codes": codes, "scale": scale.view(torch.float8_e8m0fnu)}
        y, h = add_rms_norm(t["x"], t["w"], t["r"])
        dx, dr, dw = torch.autograd.grad((y, h), (t["x"], t["r"], t["w"]), (t["dy"], t["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dr": dr, "dw": dw}
    from lockstep_amd import experts

    if c["op"] == "route":
        weights, ids = experts.route(t["logits"], c["k"], bias=t["bias"], scoring=c["scoring"], groups=c["groups"],
                                     top_groups=c["top_groups"], renormalize=c["renorm"])
        got = {"weights": weights.detach(), "experts": ids}
        if c["grad"]:
            got["dlogits"], = torch.autograd.grad(weights, t["logits"], t["dw"])
        return got
    if c["op"] == "gated":
        d = experts.dispatch(t["experts"], c["E"])
        h, scale = experts.expert_gated(t["x"], t["xs"], t["w"], t["ws"], d)
        return {"h": h, "scale": scale.view(torch.float8_e8m0fnu), "order": d.order, "offsets": d.offsets}
    d = experts.Dispatch(t["experts"], t["order"], t["offsets"])
    return experts.expert_combine(t["x"], t["xs"], t["w"], t["ws"], d, t["weights"], out_dtype=_DT[c["dtype"]])


# ------------------------------------------------------------------ its price
def work(case):
    """Bytes read and written once, and multiply-adds times two."""
    c, T = case, case["T"]
    size = 4 if c.get("dtype") == "f32" else 2
    if c["op"] == "norm":  # x and the residual in, their sum and the norm out, and its codes and scales
        return {"bytes": T * c["D"] * (4.0 * size + 33 / 32), "flops": 0.0}
    if c["op"] == "train":  # forward 2 in, 2 out; backward dy, dh and the sum in, one gradient out
        return {"bytes": 8.0 * size * T * c["D"], "flops": 0.0}
    if c["op"] == "route":
        grad = 2 * size * c["E"] + 4 * c["k"] if c["grad"] else 0
        return {"bytes": T * (size * c["E"] + 8.0 * c["k"] + grad), "flops": 0.0}
    pairs = (T - c["padded"]) * c["k"]
    # experts that some pair takes, were the pairs to choose alike
    read = c["E"] * (1 - (1 - 1 / c["E"]) ** pairs)
    if c["op"] == "gated":
        moved = read * 2 * c["F"] * c["K"] * 17 / 32 + (T * c["K"] + T * c["k"] * c["F"]) * 33 / 32
        return {"bytes": moved, "flops": 4.0 * pairs * c["K"] * c["F"]}
    moved = read * c["N"] * c["K"] * 17 / 32 + pairs * c["K"] * 33 / 32 + 2 * T * c["N"]
    return {"bytes": moved, "flops": 2.0 * pairs * c["K"] * c["N"]}


# ------------------------------------------------------------------ in 64 bits
def _grid8(x):
    """E4M3 values and scales of x [.., D] in float64."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(torch.where(top == 0, 448.0, top) / 448)).clamp(min=-127))
    r = b / s
    step = torch.exp2(torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(r / step) * step).flatten(-2), s.squeeze(-1)


def _table64(codes, scale):
    """The values of one expert's MXFP4 rows in float64."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    mag = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], device=codes.device, dtype=torch.float64) / 2
    v = mag[n & 7] * (1 - 2 * (n >> 3)).double()
    return v * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    c, op, t = case, case["op"], _inputs(case, seed)
    if op in ("norm", "train"):
        h = (t["x"].double() + t["r"].double()).to(t["x"].dtype).double()
        inv = (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        y = h * inv * t["w"].double()
        if op == "norm":
            codes, scale = _grid8(y)
            return {"y": y, "h": h, "codes": codes, "scale": scale}
        dy = t["dy"].double()
        g = dy * t["w"].double()
        dx = g * inv - h * inv ** 3 * (g * h).mean(-1, keepdim=True) + t["dh"].double()
        return {"y": y, "h": h, "dx": dx, "dr": dx, "dw": (dy * h * inv).sum(0)}
    if op == "route":
        x = t["logits"].double()
        s = torch.softmax(x, -1) if c["scoring"] == "softmax" else torch.sigmoid(x)
        rank = s.clone() if t["bias"] is None else s + t["bias"].double()
        if c["groups"] > 1:
            by = rank.view(c["T"], c["groups"], -1)
            two = by.topk(min(2, by.shape[-1]), -1).values.sum(-1)
            # a group's place: how many are larger, or as large and earlier
            n = torch.arange(c["groups"], device=x.device)
            ahead = (two[:, None] > two[..., None]) | ((two[:, None] == two[..., None]) & (n < n[:, None]))
            rank = by.masked_fill((ahead.sum(-1) >= c["top_groups"])[..., None], -math.inf).flatten(1)
        low = rank.topk(c["k"], -1).values
        at = (rank[:, None, :] == low[:, :, None]).to(torch.uint8).argmax(-1)
        tied = (low[:, 1:] == low[:, :-1]).any() or (rank >= low[:, -1:]).sum() != low.numel()
        if tied:  # of equal logits: the j-th of them for the j-th place
            at = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :c["k"]]
        a = s.gather(-1, at)
        if c["grad"]:
            x = x.requires_grad_(True)
            s = torch.softmax(x, -1) if c["scoring"] == "softmax" else torch.sigmoid(x)
            a = s.gather(-1, at)
        w = a / a.sum(-1, keepdim=True) if c["renorm"] else a
        got = {"weights": w.detach(), "experts": None}
        if c["grad"]:
            got["dlogits"], = torch.autograd.grad(w, x, t["dw"].double())
        return got
    T, k, E = c["T"], c["k"], c["E"]
    ids, x = t["experts"], t["x"].double() * torch.exp2(t["xs"].double() - 127).repeat_interleave(32, -1)
    out = torch.zeros((T, k, 2 * c["F"] if op == "gated" else c["N"]), device="cuda", dtype=torch.float64)
    for e in range(E):
        i, j = torch.nonzero(ids == e, as_tuple=True)
        if i.numel():
            out[i, j] = (x[i] if op == "gated" else x[i, j]) @ _table64(t["w"][e], t["ws"][e]).t()
    if op == "combine":
        return (out * t["weights"].double()[..., None]).sum(1)
    gate, up = out[..., :c["F"]], out[..., c["F"]:]
    h, scale = _grid8(gate * torch.sigmoid(gate) * up)
    return {"h": h, "scale": scale, "order": None, "offsets": None}

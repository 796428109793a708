"""Cases of the routed linears: products whose weight depends on the row.

Four operators, each in a plain form (elementary torch operations in f32) and,
where ``own`` is true, through the framework's entry points:

  route     top-k experts of every token, their softmax weights and the plan
            (rows sorted by expert) the grouped product runs on;
  grouped   Y[i] = act(W_e X[row_index[i]] + b_e) for the rows i of expert e,
            W the packed weights of all experts stacked;
  combine   out[t] = residual[t] + sum_j weight[t][j] Y[slot[t][j]];
  adapters  Y[i] = act(W X[i] + b + scale_a B_a (A_a X[i])), a the adapter of
            row i (or none): low-rank adapters of many requests beside one
            packed projection.

The weight a product multiplies is the packed block's decoded value rounded to
f16 (the tensor-core operand); f32 activations are staged to Q8_1 blocks first
(amax / 127 per 32 values, round half away), f16 activations are taken as they
are.
"""
import math

import torch

own = False

Q8_0, Q4_K, Q5_K, Q6_K = 8, 12, 13, 14
TYPES = {"q8_0": Q8_0, "q4_k": Q4_K, "q5_k": Q5_K, "q6_k": Q6_K}
ROW_BYTES = {"q8_0": 34 / 32, "q4_k": 144 / 256, "q5_k": 176 / 256, "q6_k": 210 / 256}
ELEMENT = {"f16": 2, "f32": 4}


def listed():
    return [
        # The router of one decoding step of a small batch.
        {"name": "route_decode", "op": "route", "tokens": 32, "experts": 64, "top_k": 6, "normalize": True,
         "masked": 0.0},
        # The router of a long prefill over many experts, some of them masked per token.
        {"name": "route_prefill", "op": "route", "tokens": 16384, "experts": 128, "top_k": 8, "normalize": False,
         "masked": 0.1},
        # One token through two of eight experts of the text MLP's width: latency.
        {"name": "grouped_token", "op": "grouped", "weights": "q8_0", "k": 1024, "n": 4096, "experts": 8, "tokens": 1,
         "top_k": 2, "gather": True, "skew": 0.0, "x": "f16", "y": "f16", "gelu": True},
        # A decoding batch that wakes every expert: the packed weights are the traffic.
        {"name": "grouped_decode", "op": "grouped", "weights": "q4_k", "k": 1024, "n": 4096, "experts": 32,
         "tokens": 128, "top_k": 2, "gather": True, "skew": 0.5, "x": "f16", "y": "f16", "gelu": True},
        # Many narrow experts (the fusion FFN's widths) under skewed routing: ragged groups, some empty.
        {"name": "grouped_narrow", "op": "grouped", "weights": "q6_k", "k": 256, "n": 2048, "experts": 64,
         "tokens": 777, "top_k": 1, "gather": False, "skew": 1.5, "x": "f16", "y": "f32", "gelu": False},
        # One image's tokens through the vision MLP's first product, two experts each.
        {"name": "grouped_up", "op": "grouped", "weights": "q8_0", "k": 1024, "n": 4736, "experts": 8, "tokens": 5184,
         "top_k": 2, "gather": True, "skew": 0.5, "x": "f16", "y": "f16", "gelu": True},
        # The second product of the same MLP from f32 activations (staged).
        {"name": "grouped_down", "op": "grouped", "weights": "q8_0", "k": 4736, "n": 1024, "experts": 8,
         "tokens": 5184, "top_k": 2, "gather": False, "skew": 0.5, "x": "f32", "y": "f32", "gelu": False},
        # The sum back into the residual stream, decoding and prefill.
        {"name": "combine_decode", "op": "combine", "tokens": 32, "top_k": 2, "width": 1024, "y": "f16",
         "residual": True, "dropped": 0.0},
        {"name": "combine_prefill", "op": "combine", "tokens": 16384, "top_k": 8, "width": 1024, "y": "f16",
         "residual": True, "dropped": 0.05},
        # Sixteen decoding requests, each with its own adapter.
        {"name": "adapters_decode", "op": "adapters", "weights": "q4_k", "k": 1024, "n": 4096, "m": 16, "rank": 16,
         "adapters": 16, "segments": 16, "without": 0.1, "x": "f16", "y": "f16", "gelu": False},
        # A mixed batch of short requests from f32 activations.
        {"name": "adapters_batch", "op": "adapters", "weights": "q8_0", "k": 1024, "n": 1024, "m": 250, "rank": 24,
         "adapters": 32, "segments": 100, "without": 0.2, "x": "f32", "y": "f32", "gelu": False},
        # Four requests' prefill through the vision MLP's first product.
        {"name": "adapters_prefill", "op": "adapters", "weights": "q8_0", "k": 1024, "n": 4736, "m": 5184, "rank": 64,
         "adapters": 4, "segments": 4, "without": 0.0, "x": "f16", "y": "f16", "gelu": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "grouped", "grouped", "combine", "adapters", "adapters"])
    if op == "route":
        experts = _log_int(rng, 2, 128)
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "experts": experts,
                "top_k": rng.randint(1, min(8, experts)), "normalize": rng.random() < 0.5,
                "masked": rng.choice([0.0, 0.1, 0.6])}
    if op == "combine":
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "top_k": rng.randint(1, 8),
                "width": rng.choice([256, 1000, 1024]), "y": rng.choice(["f16", "f32"]) if rng.random() < 0.5 else "f16",
                "residual": rng.random() < 0.7, "dropped": rng.choice([0.0, 0.05])}
    weights = rng.choice(["q8_0", "q4_k", "q5_k", "q6_k"])
    k = rng.choice([256, 1024, 2048]) if weights != "q8_0" else rng.choice([96, 256, 1024, 2080])
    n = rng.choice([200, 256, 1000, 1024, 2048, 4096])
    types = {"x": rng.choice(["f16", "f32"]), "y": rng.choice(["f16", "f32"]), "gelu": rng.random() < 0.5}
    if op == "grouped":
        top_k = rng.randint(1, 2)
        return {"op": op, "weights": weights, "k": k, "n": n, "experts": _log_int(rng, 1, 16),
                "tokens": _log_int(rng, 1, 4000), "top_k": top_k, "gather": top_k > 1 or rng.random() < 0.5,
                "skew": rng.choice([0.0, 0.5, 1.5]), **types}
    m = _log_int(rng, 1, 4000)
    return {"op": op, "weights": weights, "k": k, "n": n, "m": m, "rank": _log_int(rng, 1, 128),
            "adapters": _log_int(rng, 1, 24), "segments": _log_int(rng, 1, m), "without": rng.choice([0.0, 0.2]),
            **types}


# ---- inputs ---------------------------------------------------------------------

def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _packed(g, kind, n, k):
    """GGUF rows [n][row bytes] (uint8) of weights near N(0, 0.02^2), and their decoded f32 values [n][k]."""
    if kind == "q8_0":
        w = _normal(g, n, k // 32, 32) * 0.02
        d = (w.abs().amax(-1, keepdim=True) / 127).half()
        q = torch.round(w / d.float()).clamp_(-127, 127)
        rows = torch.cat([d.view(torch.uint8), q.to(torch.int8).view(torch.uint8)], -1)
        return rows.reshape(n, -1), (q * d.float()).reshape(n, k)
    blocks = n * (k // 256)
    if kind == "q6_k":
        q = (32 + 9 * _normal(g, blocks, 256)).round_().clamp_(0, 63).to(torch.int32)
        sc = torch.randint(40, 100, (blocks, 16), generator=g, device="cuda", dtype=torch.int32)
        d = (0.02 / (9 * 70) * (0.8 + 0.4 * _rand(g, blocks, 1))).half()
        parts = q.view(blocks, 2, 4, 32)  # half, quarter, position
        ql = torch.cat([(parts[:, :, 0] & 15) | ((parts[:, :, 2] & 15) << 4),
                        (parts[:, :, 1] & 15) | ((parts[:, :, 3] & 15) << 4)], -1)
        qh = (parts[:, :, 0] >> 4) | (parts[:, :, 1] >> 4 << 2) | (parts[:, :, 2] >> 4 << 4) | (parts[:, :, 3] >> 4 << 6)
        rows = torch.cat([ql.reshape(blocks, 128).to(torch.uint8), qh.reshape(blocks, 64).to(torch.uint8),
                          sc.to(torch.uint8), d.view(torch.uint8)], -1)
        w = (d.float() * sc.float()).repeat_interleave(16, -1) * (q - 32).float()
        return rows.reshape(n, -1), w.reshape(n, k)
    top, mid, sd = (15, 7.5, 2.6) if kind == "q4_k" else (31, 15.5, 5.2)
    q = (mid + sd * _normal(g, blocks, 8, 32)).round_().clamp_(0, top).to(torch.int32)
    sc = torch.randint(32, 62, (blocks, 8), generator=g, device="cuda", dtype=torch.int32)
    mn = sc + torch.randint(-1, 2, (blocks, 8), generator=g, device="cuda", dtype=torch.int32)
    d = (0.02 / (sd * 47) * (0.8 + 0.4 * _rand(g, blocks, 1))).half()
    dmin = (d.float() * mid).half()
    scales = torch.cat([sc[:, :4] | (sc[:, 4:] >> 4 << 6), mn[:, :4] | (mn[:, 4:] >> 4 << 6),
                        (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)], -1).to(torch.uint8)
    pair = q.view(blocks, 4, 2, 32) & 15
    qs = (pair[:, :, 0] | (pair[:, :, 1] << 4)).reshape(blocks, 128).to(torch.uint8)
    high = [] if kind == "q4_k" else [((q >> 4) << torch.arange(8, device="cuda").view(1, 8, 1)).sum(1).to(torch.uint8)]
    rows = torch.cat([d.view(torch.uint8), dmin.view(torch.uint8), scales, *high, qs], -1)
    w = (d.float() * sc.float()).unsqueeze(-1) * q.float() - (dmin.float() * mn.float()).unsqueeze(-1)
    return rows.reshape(n, -1), w.reshape(n, k)


def _dtype(name):
    return torch.float16 if name == "f16" else torch.float32


def _activations(g, rows, k, kind):
    """LayerNorm-like rows with a few large channels."""
    x = _normal(g, rows, k)
    x[:, :: 97] *= 4
    return x.to(_dtype(kind))


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "route":
        t, e = case["tokens"], case["experts"]
        logits = _normal(g, t, e) + 0.5 * _normal(g, 1, e)
        logits = torch.round(logits * 256) / 256  # router logits of 16-bit activations: ties happen
        logits[_rand(g, t, e) < case["masked"]] = -math.inf
        s["logits"] = logits
        return s
    if op == "combine":
        t, j, w = case["tokens"], case["top_k"], case["width"]
        s["y"] = _normal(g, t * j, w).to(_dtype(case["y"]))
        slots = torch.randperm(t * j, generator=g, device="cuda").to(torch.int32).view(t, j)
        slots[_rand(g, t, j) < case["dropped"]] = -1
        s["slots"] = slots
        weights = _rand(g, t, j) + 0.05
        s["weights"] = weights / weights.sum(1, keepdim=True)
        s["residual"] = _normal(g, t, w) if case["residual"] else None
        return s
    k, n = case["k"], case["n"]
    count = case["experts"] if op == "grouped" else 1
    s["gguf"], s["w32"] = _packed(g, case["weights"], count * n, k)
    s["bias"] = 0.1 * _normal(g, count * n)
    if op == "grouped":
        tokens, e = case["tokens"], count
        popularity = torch.exp(case["skew"] * _normal(g, e)) + 1e-6
        top_k = min(case["top_k"], e)
        # top_k distinct experts a token (without replacement, by perturbed log popularity)
        keys = popularity.log() - (-_rand(g, tokens, e).clamp_min(1e-12).log()).log()
        choice = keys.topk(top_k, 1).indices
        flat, order = choice.reshape(-1).sort(stable=True)
        rows = tokens * top_k
        s["offsets"] = torch.searchsorted(flat, torch.arange(e + 1, device="cuda")).to(torch.int32)
        s["expert"] = flat
        s["row_index"] = (order // top_k).to(torch.int32) if case["gather"] else None
        s["rows"] = rows
        s["x"] = _activations(g, tokens if case["gather"] else rows, k, case["x"])
        return s
    m, r, count = case["m"], case["rank"], case["adapters"]
    s["x"] = _activations(g, m, k, case["x"])
    s["a"] = (_normal(g, count, r, k) / math.sqrt(k)).half()
    s["b"] = (_normal(g, count, n, r) * 0.1).half()
    s["scale"] = 0.5 + _rand(g, count)
    cuts = torch.randperm(max(m - 1, 1), generator=g, device="cuda")[: min(case["segments"], m) - 1] + 1
    start = torch.zeros(m, device="cuda", dtype=torch.int64)
    start[cuts[cuts < m]] = 1
    segment = start.cumsum(0)
    owner = torch.randint(0, count, (m,), generator=g, device="cuda")
    owner[_rand(g, m) < case["without"]] = -1
    s["ids"] = owner[segment].to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        new = lambda shape, dtype: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
        s["out"] = {"weights": new((t, k), torch.float32), "ids": new((t, k), torch.int32),
                    "offsets": new((e + 1,), torch.int32), "rows": new((t * k,), torch.int32),
                    "slots": new((t, k), torch.int32)}
        if own:
            samq = _samq()
            s["workspace"] = _workspace(samq.route_workspace(t, e, k))
        return s
    if op == "combine":
        s["out"] = torch.empty(case["tokens"], case["width"], device="cuda")
        if own:
            _samq()
        return s
    gguf, w32 = s.pop("gguf"), s.pop("w32")
    n, k = case["n"], case["k"]
    rows = s["rows"] if op == "grouped" else case["m"]
    s["y"] = torch.empty(rows, n, device="cuda", dtype=_dtype(case["y"]))
    if op == "grouped":
        # what a plan of padded groups keeps: each row's place in its group, the largest group
        first = s["offsets"][:-1].long()
        s["place"] = torch.arange(rows, device="cuda") - first[s["expert"]]
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    else:
        order = torch.argsort(s["ids"], stable=True)
        ids = s["ids"][order].long()
        has = ids >= 0
        s["order"], s["owner"] = order[has], ids[has]
        first = torch.searchsorted(s["owner"], torch.arange(case["adapters"], device="cuda"))
        s["place"] = torch.arange(s["owner"].numel(), device="cuda") - first[s["owner"]]
        s["most"] = max(1, int(torch.bincount(s["owner"], minlength=1).max()) if s["owner"].numel() else 1)
    if own:
        samq = _samq()
        s["handle"] = samq.Weights(TYPES[case["weights"]], k, gguf.shape[0], gguf.cpu().numpy())
        if op == "grouped":
            s["workspace"] = _workspace(samq.linear_grouped_workspace(s["handle"], case["experts"], s["x"].shape[0], rows,
                                                                      s["x"].dtype))
        else:
            s["adapters"] = samq.Adapters(k, n, case["rank"], case["adapters"])
            a, b, scale = s["a"].cpu().numpy(), s["b"].cpu().numpy(), s["scale"].tolist()
            for i in range(case["adapters"]):
                s["adapters"].set(i, a[i], b[i], scale[i])
            s["workspace"] = _workspace(samq.linear_adapters_workspace(s["handle"], s["adapters"], rows, s["x"].dtype))
    else:
        s["w"] = w32.half().float().view(-1, n, k)
    return s


def _workspace(size):
    return torch.empty(size, device="cuda", dtype=torch.uint8) if size else None


def _samq():
    import os
    import sys
    package = os.path.join(os.getcwd(), "sam.cpp_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import samq
    return samq


# ---- one pass ----------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"route": _route, "combine": _combine, "grouped": _grouped, "adapters": _adapters}[state["case"]["op"]](state)


def _run_own(s):
    import samq
    c, op = s["case"], s["case"]["op"]
    if op == "route":
        o = s["out"]
        samq.route(s["logits"], c["tokens"], c["experts"], c["experts"], c["top_k"], o["weights"], o["ids"],
                   o["offsets"], o["rows"], o["slots"], normalize=c["normalize"], workspace=s["workspace"])
        return o
    if op == "combine":
        rows, width = s["y"].shape
        samq.combine(s["y"], rows, width, s["slots"], s["weights"], c["tokens"], c["top_k"], width, s["out"], width,
                     residual=s["residual"], ldr=width)
        return s["out"]
    epilogue = samq.EPILOGUE_GELU_ERF if c["gelu"] else samq.EPILOGUE_NONE
    x = s["x"]
    if op == "grouped":
        samq.linear_grouped(s["handle"], c["experts"], x, x.shape[0], c["k"], s["offsets"], s["rows"], s["y"], c["n"],
                            row_index=s["row_index"], bias=s["bias"], epilogue=epilogue, workspace=s["workspace"])
    else:
        samq.linear_adapters(s["handle"], s["adapters"], x, c["m"], c["k"], s["ids"], s["y"], c["n"], bias=s["bias"],
                             epilogue=epilogue, workspace=s["workspace"])
    return s["y"]


def _stage(x):
    """The f32 values of the product's activation operand: f16 as it is, f32 through Q8_1 blocks of 32."""
    if x.dtype == torch.float16:
        return x.float()
    v = x.view(x.shape[0], -1, 32)
    amax = v.abs().amax(-1, keepdim=True)
    # quotients of two tensors: torch turns one by or of a Python number into a product with a rounded reciprocal
    top = torch.full_like(amax, 127)
    d = (amax / top).half().float()
    t = v.abs() * torch.where(amax == 0, torch.zeros_like(amax), top / amax)
    whole = t.trunc()
    q = torch.copysign(whole + (t - whole >= 0.5), v)
    return (d * q).half().float().view(x.shape)


def _gelu(v):
    return 0.5 * v * (1 + torch.erf(v * 0.7071067811865476))


def _padded(x, owner, place, count, most):
    """Rows of x in their places of [count][most] padded groups."""
    out = torch.zeros(count, most, x.shape[1], device=x.device, dtype=x.dtype)
    out[owner, place] = x
    return out


def _grouped(s):
    c, x = s["case"], _stage(s["x"])
    if s["row_index"] is not None:
        x = x[s["row_index"].long()]
    e = c["experts"]
    y = torch.bmm(_padded(x, s["expert"], s["place"], e, s["most"]), s["w"].transpose(1, 2))
    y = y + s["bias"].view(e, 1, -1)
    y = y[s["expert"], s["place"]]
    if c["gelu"]:
        y = _gelu(y)
    s["y"].copy_(y)
    return s["y"]


def _adapters(s):
    c, x = s["case"], _stage(s["x"])
    y = x @ s["w"][0].t() + s["bias"]
    owned = _padded(x[s["order"]], s["owner"], s["place"], c["adapters"], s["most"])
    h = torch.bmm(owned, s["a"].float().transpose(1, 2)) * s["scale"].view(-1, 1, 1)
    delta = torch.bmm(h, s["b"].float().transpose(1, 2))
    y[s["order"]] += delta[s["owner"], s["place"]]
    if c["gelu"]:
        y = _gelu(y)
    s["y"].copy_(y)
    return s["y"]


def _combine(s):
    y, slots = s["y"].float(), s["slots"].long()
    keep = (slots >= 0).unsqueeze(-1)
    terms = torch.where(keep, y[slots.clamp_min(0)] * s["weights"].unsqueeze(-1), torch.zeros((), device=y.device))
    out = terms.sum(1)
    if s["residual"] is not None:
        out = out + s["residual"]
    s["out"].copy_(out)
    return s["out"]


def _route(s):
    c, o = s["case"], s["out"]
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    logits = torch.where(torch.isfinite(s["logits"]), s["logits"], torch.full((), -math.inf, device="cuda"))
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)  # ties: the lowest index first
    top, ids = value[:, :k], index[:, :k]
    taken = torch.isfinite(top)
    best = torch.where(taken[:, :1], top[:, :1], torch.zeros_like(top[:, :1]))
    p = torch.exp(top - best)
    total = p.sum(1, keepdim=True) if c["normalize"] else torch.exp(value - best).sum(1, keepdim=True)
    o["weights"].copy_(torch.where(taken, p / total, torch.zeros_like(p)))
    ids = torch.where(taken, ids, torch.full_like(ids, -1))
    o["ids"].copy_(ids)
    flat = torch.where(ids < 0, torch.full_like(ids, e), ids).reshape(-1)
    order = torch.argsort(flat, stable=True)
    counts = torch.zeros(e + 1, device="cuda", dtype=torch.int64).scatter_add_(0, flat, torch.ones_like(flat))
    ends = counts.cumsum(0)
    o["offsets"][0] = 0
    o["offsets"][1:].copy_(ends[:e])
    at = torch.arange(t * k, device="cuda")
    o["rows"].copy_(torch.where(at < ends[e - 1], order // k, torch.full_like(order, -1)))
    slots = torch.empty_like(order)
    slots[order] = at
    o["slots"].copy_(torch.where(flat < e, slots, torch.full_like(slots, -1)).view(t, k))
    return o


# ---- work ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": 4 * t * e + 16 * t * k + 4 * (e + 1), "flops": 4 * t * e}
    if op == "combine":
        t, j, w = case["tokens"], case["top_k"], case["width"]
        kept = t * j * (1 - case["dropped"])
        return {"bytes": kept * w * ELEMENT[case["y"]] + 8 * t * j + 4 * t * w * (2 if case["residual"] else 1),
                "flops": 2 * kept * w}
    k, n = case["k"], case["n"]
    packed = ROW_BYTES[case["weights"]] * k * n
    if op == "grouped":
        e = case["experts"]
        rows = case["tokens"] * min(case["top_k"], e)
        read = case["tokens"] if case["gather"] else rows
        awake = min(e, rows)
        return {"bytes": awake * (packed + 4 * n) + read * k * ELEMENT[case["x"]] + rows * n * ELEMENT[case["y"]] +
                4 * (e + 1) + (4 * rows if case["gather"] else 0), "flops": 2 * rows * n * k}
    m, r = case["m"], case["rank"]
    awake = min(case["adapters"], case["segments"], m)
    with_one = m * (1 - case["without"])
    return {"bytes": packed + 4 * n + 2 * awake * r * (k + n) + m * k * ELEMENT[case["x"]] +
            m * n * ELEMENT[case["y"]] + 4 * m, "flops": 2 * m * n * k + 2 * with_one * r * (k + n)}


# ---- the definition in 64 bits ----------------------------------------------------------

def _decoded64(gguf, kind, k):
    """f16 operand values (as f64) of GGUF rows, from the bytes."""
    rows = gguf.shape[0]
    def scalar(b):
        return b.contiguous().view(torch.float16).double()
    if kind == "q8_0":
        b = gguf.view(rows, -1, 34)
        w = scalar(b[..., :2]) * b[..., 2:].contiguous().view(torch.int8).double()
    elif kind == "q6_k":
        b = gguf.view(-1, 210)
        low, high, sc, d = b[:, :128].int(), b[:, 128:192].int(), b[:, 192:208].contiguous().view(torch.int8), b[:, 208:]
        e = torch.arange(256, device=b.device)
        half, quarter, pos = e // 128, e % 128 // 32, e % 32
        nibble = low[:, half * 64 + (quarter % 2) * 32 + pos] >> (4 * (quarter // 2)) & 15
        two = high[:, half * 32 + pos] >> (2 * quarter) & 3
        w = scalar(d) * sc.double()[:, e // 16] * (nibble + 16 * two - 32).double()
    else:
        size = 144 if kind == "q4_k" else 176
        b = gguf.view(-1, size)
        packed, codes = b[:, 4:16].int(), b[:, size - 128:].int()
        e = torch.arange(256, device=b.device)
        sub, pos = e // 32, e % 32
        q = codes[:, sub // 2 * 32 + pos] >> (4 * (sub % 2)) & 15
        if kind == "q5_k":
            q = q + 16 * (b[:, 16:48].int()[:, pos] >> sub & 1)
        j = torch.arange(8, device=b.device)
        first = j < 4
        sc = torch.where(first, packed[:, j] & 63, (packed[:, (j + 4).clamp_max(11)] & 15) | (packed[:, (j - 4).clamp_min(0)] >> 6 << 4))
        mn = torch.where(first, packed[:, (j + 4).clamp_max(11)] & 63, (packed[:, (j + 4).clamp_max(11)] >> 4) | (packed[:, j] >> 6 << 4))
        w = scalar(b[:, :2]) * sc.double()[:, sub] * q.double() - scalar(b[:, 2:4]) * mn.double()[:, sub]
    return w.reshape(rows, k).half().double()


def _operand64(x):
    """The activation operand. A Q8_1 block's scale and codes are whole steps of f32 arithmetic by definition."""
    if x.dtype == torch.float16:
        return x.double()
    blocks = x.reshape(-1, 32)
    peak = blocks.abs().max(1, keepdim=True).values
    step = (peak.double() / 127).float().half().double()
    scaled = blocks * torch.where(peak > 0, (127 / peak.double()).float(), peak)
    code = torch.floor(scaled.double().abs() + 0.5) * torch.sign(scaled.double())
    return (step * code).half().double().reshape(x.shape)


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "route":
        z = s["logits"].double()
        z = z.masked_fill(~torch.isfinite(z), -math.inf)
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        left, ids, vals = z.clone(), [], []
        for _ in range(k):  # the lowest index among the largest
            v = left.max(1, keepdim=True).values
            i = torch.where(left == v, torch.arange(e, device=z.device), e).min(1, keepdim=True).values
            ids.append(torch.where(torch.isfinite(v), i, torch.full_like(i, -1)))
            vals.append(v)
            left.scatter_(1, i, -math.inf)
        ids, vals = torch.cat(ids, 1), torch.cat(vals, 1)
        base = vals if case["normalize"] else z
        p = torch.exp(vals - torch.logsumexp(base, 1, keepdim=True))
        p = torch.where(ids >= 0, p, torch.zeros_like(p))
        flat = ids.reshape(-1).cpu()
        offsets, rows, slots = [0], [], torch.full((t * k,), -1, dtype=torch.int64)
        for i in range(e):
            mine = (flat == i).nonzero().view(-1)
            slots[mine] = torch.arange(mine.numel()) + offsets[-1]
            rows.append(mine // k)
            offsets.append(offsets[-1] + mine.numel())
        rows = torch.cat(rows + [torch.full((t * k - offsets[-1],), -1, dtype=torch.int64)])
        return {"weights": p, "ids": ids.int(), "offsets": torch.tensor(offsets, dtype=torch.int32),
                "rows": rows.int(), "slots": slots.view(t, k).int()}
    if op == "combine":
        out = torch.zeros(case["tokens"], case["width"], device="cuda", dtype=torch.float64)
        if s["residual"] is not None:
            out += s["residual"].double()
        for j in range(case["top_k"]):
            at = s["slots"][:, j].long()
            have = (at >= 0).nonzero().view(-1)
            out[have] += s["weights"][have, j, None].double() * s["y"][at[have]].double()
        return out
    n, k = case["n"], case["k"]
    w = _decoded64(s["gguf"], case["weights"], k)
    del s["gguf"], s["w32"]
    x, bias = _operand64(s["x"]), s["bias"].double()
    if op == "grouped":
        y = torch.empty(s["rows"], n, device="cuda", dtype=torch.float64)
        cut = s["offsets"].tolist()
        for e in range(case["experts"]):
            lo, hi = cut[e], cut[e + 1]
            at = torch.arange(lo, hi, device="cuda") if s["row_index"] is None else s["row_index"][lo:hi].long()
            y[lo:hi] = x[at] @ w[e * n:(e + 1) * n].t() + bias[e * n:(e + 1) * n]
    else:
        y = x @ w.t() + bias
        for a in range(case["adapters"]):
            mine = (s["ids"] == a).nonzero().view(-1)
            y[mine] += s["scale"][a].double() * ((x[mine] @ s["a"][a].double().t()) @ s["b"][a].double().t())
    return y * torch.special.ndtr(y) if case["gelu"] else y

"""The routed linears on the GPU (samq_route_v1, samq_linear_grouped_v1,
samq_combine_v1, samq_linear_adapters_v1) against plain 64-bit definitions.

Tolerances, per output and from arithmetic alone.  The operands are exact (f16
weights and activations), so a product of depth k differs from the 64-bit one by
the f32 accumulation: a 16-deep step of the tensor core adds its exact products
to the accumulator with one truncation, so at most k / 16 + 8 additions off by
2^-23 of the running magnitude, itself at most sum |w x|.  Then one rounding of
the output: half a step, 2^-24 (f32) or 2^-11 (f16, 2^-25 below its normal
range) of the value.  The erf-GELU polynomial is within 1.5e-7 of |x| / 2 and its
two approximate functions within 2^-22 each; its slope is at most 1.13.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

Q8_0, Q4_K, Q5_K, Q6_K = 8, 12, 13, 14
SENTINEL = -77.0


@pytest.fixture(scope="module")
def samq():
    import samq as module
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    module.init(0)
    return module


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def erf_gelu64(v):
    return np.array([0.5 * x * math.erfc(-x / math.sqrt(2.0)) for x in v.ravel()]).reshape(v.shape)


def packed(oracle, rng, qtype, n, k):
    w = rng.normal(0, 0.02, (n, k)).astype(np.float32)
    w[rng.random(w.shape) < 0.01] *= 8
    rows = oracle.quantize(qtype, w)
    return rows, oracle.weight_f16(qtype, k, n, rows).astype(np.float64)


def operand64(oracle, x):
    """The product's activation operand as f64: f16 as it is, f32 staged to Q8_1."""
    if x.dtype == np.float16:
        return x.astype(np.float64)
    return oracle.act_f16(np.ascontiguousarray(x)).astype(np.float64)


def accumulation(k, magnitude):
    return (k / 16 + 8) * 2.0 ** -23 * magnitude


def finished(pre, tol, gelu, dtype):
    """(reference, tolerance) after the epilogue and the output's rounding."""
    ref = erf_gelu64(pre) if gelu else pre
    if gelu:
        tol = 1.13 * tol + (1.5e-7 / 2 + 2.0 ** -21) * np.abs(pre)
    half = 2.0 ** -11 if dtype == np.float16 else 2.0 ** -24
    return ref, tol + half * (np.abs(ref) + tol) + (2.0 ** -25 if dtype == np.float16 else 2.0 ** -149)


def assert_close(got, ref, tol, what=""):
    off = np.abs(got.astype(np.float64) - ref)
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(off / tol)))


# ---- router -------------------------------------------------------------------

def route_reference(logits, top_k, normalize):
    t, e = logits.shape
    z = np.where(np.isfinite(logits), logits.astype(np.float64), -np.inf)
    order = np.argsort(-z, axis=1, kind="stable")[:, :top_k]
    val = np.take_along_axis(z, order, 1)
    taken = np.isfinite(val)
    ids = np.where(taken, order, -1)
    weights = np.zeros((t, top_k))
    for i in range(t):
        if taken[i].any():
            p = np.where(taken[i], np.exp(val[i] - val[i, 0], where=taken[i], out=np.zeros(top_k)), 0)
            rest = z[i][np.isfinite(z[i])]
            weights[i] = p / (p.sum() if normalize else np.exp(rest - val[i, 0]).sum())
    flat = ids.reshape(-1)
    offsets = np.zeros(e + 1, np.int64)
    rows = np.full(t * top_k, -1, np.int64)
    slots = np.full(t * top_k, -1, np.int64)
    at = 0
    for x in range(e):
        offsets[x] = at
        for i in np.nonzero(flat == x)[0]:
            rows[at] = i // top_k
            slots[i] = at
            at += 1
    offsets[e] = at
    return weights, ids, offsets, rows, slots.reshape(t, top_k)


def run_route(samq, logits, top_k, normalize, ld=None, workspace=True):
    t, e = logits.shape
    ld = ld or e
    full = np.full((max(t, 1), ld), 9e9, np.float32)
    full[:t, :e] = logits
    new = lambda n: torch.full((max(n, 1),), 12345, dtype=torch.int32, device="cuda")  # noqa: E731
    w = torch.full((max(t * top_k, 1),), SENTINEL, device="cuda")
    ids, offsets, rows, slots = new(t * top_k), new(e + 1), new(t * top_k), new(t * top_k)
    space = torch.full((samq.route_workspace(t, e, top_k),), 255, dtype=torch.uint8, device="cuda")
    samq.route(dev(full), t, e, ld, top_k, w, ids, offsets, rows, slots, normalize=normalize,
               workspace=space if workspace else None)
    n = t * top_k
    return (host(w)[:n].reshape(t, top_k), host(ids)[:n].reshape(t, top_k), host(offsets), host(rows)[:n],
            host(slots)[:n].reshape(t, top_k))


@pytest.mark.parametrize("tokens,experts,top_k,masked,normalize,ld", [
    (0, 8, 2, 0.0, True, None), (1, 1, 1, 0.0, True, None), (1, 8, 2, 0.0, False, 9), (31, 7, 7, 0.3, True, None),
    (64, 64, 6, 0.0, True, None), (65, 64, 6, 0.9, False, 67), (300, 100, 8, 0.5, True, None),
    (1000, 129, 3, 0.0, False, None), (700, 257, 32, 0.2, True, 300), (50, 1000, 32, 0.97, True, None),
    (5000, 33, 4, 0.1, False, None), (40000, 16, 2, 0.0, True, None), (9000, 3, 1, 0.99, True, None),
    (700, 1024, 8, 0.0, False, None), (64, 128, 32, 0.4, False, 130)])
def test_route(samq, tokens, experts, top_k, masked, normalize, ld):
    rng = np.random.default_rng(tokens * 31 + experts)
    logits = (np.round(rng.normal(0, 1.5, (tokens, experts)) * 16) / 16).astype(np.float32)  # many ties
    logits[rng.random(logits.shape) < masked] = -np.inf
    if tokens > 4 and experts > 2:
        logits[1] = -np.inf             # a row with nothing eligible
        logits[2, 1] = np.nan
        logits[3, 0] = np.inf           # not eligible either
        logits[4] = np.finfo(np.float32).min  # the type's lowest value is an ordinary logit
    got = run_route(samq, logits, top_k, normalize, ld)
    ref = route_reference(logits, top_k, normalize)
    for name, g, r in zip(("ids", "offsets", "rows", "slots"), got[1:], ref[1:]):
        np.testing.assert_array_equal(g, r, err_msg=name)
    # expf within 2 ulp of each term, the f32 argument's rounding (2^-24 |l - max|, at most 110 where exp is not yet
    # zero in f32), the sum of the experts' terms and the quotient; below f32's normal range 2^-126
    tol = (2 * 110 + experts + 8) * 2.0 ** -24
    assert_close(got[0], ref[0], tol * ref[0] + 2.0 ** -126, "weights")


def test_route_is_repeatable(samq):
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 1, (3000, 40)).astype(np.float32)
    first = run_route(samq, logits, 4, True)
    for _ in range(3):
        for a, b in zip(first, run_route(samq, logits, 4, True, workspace=False)):
            np.testing.assert_array_equal(a, b)


# ---- grouped products -----------------------------------------------------------

def grouped_case(samq, oracle, qtype, k, n, sizes, x_dtype, y_dtype, gelu, gather, bias=True, lead=0, tail=0,
                 pad_x=0, pad_y=0, seed=0, poison=None):
    """Runs one grouped product and its reference; returns (y with padding, reference, tolerance, lead)."""
    rng = np.random.default_rng(seed + 7 * k + n)
    groups = len(sizes)
    gguf, w = packed(oracle, rng, qtype, groups * n, k)
    total = int(np.sum(sizes))
    rows = lead + total + tail
    offsets = (lead + np.concatenate([[0], np.cumsum(sizes)])).astype(np.int32)
    x_rows = max(1, total // 2) if gather else rows
    unit_x, unit_y = (8 if x_dtype == np.float16 else 4), (8 if y_dtype == np.float16 else 4)
    ldx = (k + unit_x - 1) // unit_x * unit_x + pad_x * unit_x
    ldy = (n + unit_y - 1) // unit_y * unit_y + pad_y * unit_y
    x = np.full((x_rows, ldx), 1e4, x_dtype)
    x[:, :k] = rng.normal(0, 1, (x_rows, k))
    if poison is not None:
        poison(x)
    index = rng.integers(0, x_rows, rows).astype(np.int32) if gather else None
    if gather and total > 3:
        index[lead + 1] = -1
        index[lead + 2] = x_rows
    b = rng.normal(0, 0.3, (groups, n)).astype(np.float32) if bias else None
    weights = samq.Weights(qtype, k, groups * n, gguf)
    y = torch.full((rows, ldy), SENTINEL, dtype=torch.float16 if y_dtype == np.float16 else torch.float32,
                   device="cuda")
    space = samq.linear_grouped_workspace(weights, groups, x_rows, rows, torch.float16 if x_dtype == np.float16
                                          else torch.float32)
    samq.linear_grouped(weights, groups, dev(x), x_rows, ldx, dev(offsets), rows, y, ldy,
                        row_index=None if index is None else dev(index), bias=None if b is None else dev(b),
                        epilogue=1 if gelu else 0,
                        workspace=torch.full((space,), 255, dtype=torch.uint8, device="cuda") if space else None)
    got = host(y)
    weights.close()
    xo = operand64(oracle, x[:, :k])
    pre = np.zeros((total, n))
    mag = np.zeros((total, n))
    for g in range(groups):
        lo, hi = offsets[g] - lead, offsets[g + 1] - lead
        src = np.arange(lo, hi) + lead if index is None else index[lo + lead:hi + lead]
        ok = (src >= 0) & (src < x_rows)
        xs = np.where(ok[:, None], xo[np.clip(src, 0, x_rows - 1)], 0.0)
        wg = w[g * n:(g + 1) * n]
        pre[lo:hi] = xs @ wg.T + (b[g] if bias else 0.0)
        mag[lo:hi] = np.abs(xs) @ np.abs(wg).T + (np.abs(b[g]) if bias else 0.0)
    ref, tol = finished(pre, accumulation(k, mag), gelu, y_dtype)
    inside = slice(lead, lead + total)
    assert (got[:lead] == SENTINEL).all() and (got[lead + total:] == SENTINEL).all(), "rows outside every group changed"
    assert (got[inside, n:] == SENTINEL).all(), "columns behind n changed"
    return got[inside, :n], ref, tol


H, F = np.float16, np.float32


@pytest.mark.parametrize("qtype,k,n,sizes,x_dtype,y_dtype,gelu,gather,extra", [
    (Q8_0, 32, 8, [1], H, F, False, False, {}),
    (Q8_0, 96, 201, [3, 0, 1], H, H, False, False, {"pad_y": 1}),
    (Q4_K, 256, 128, [1, 1], H, H, True, True, {}),
    (Q5_K, 512, 136, [0, 0, 5, 0], F, F, False, False, {"pad_x": 2}),
    (Q6_K, 256, 264, [16, 17, 15, 0, 33], H, F, True, False, {"lead": 3, "tail": 5}),
    (Q8_0, 160, 72, [64, 65, 63, 1], F, H, False, True, {"pad_x": 1, "pad_y": 2}),
    (Q4_K, 768, 320, [127, 0, 129, 128], H, H, False, False, {"tail": 1}),
    (Q8_0, 1056, 384, [300, 2, 0, 41], H, F, True, True, {"lead": 1, "pad_x": 3}),
    (Q5_K, 1024, 200, [257, 511, 1, 90], H, H, True, False, {"bias": False}),
    (Q6_K, 512, 1000, [700, 0, 0, 30], F, F, False, True, {"lead": 2, "tail": 2}),
    (Q8_0, 4736, 264, [70, 5], H, F, False, False, {"bias": False}),
    (Q4_K, 1024, 520, [0, 0, 0], H, H, False, False, {"tail": 4}),
    (Q8_0, 64, 16, [2] * 200, H, H, False, True, {}),
    (Q8_0, 1024, 256, [1500], H, H, True, False, {"tail": 7}),
    (Q4_K, 256, 640, [5, 1100, 64], F, H, True, True, {}),
    (Q8_0, 64, 40, [70, 3] * 100, H, F, False, True, {"lead": 1, "tail": 1}),   # both kernels, over 128 groups
    (Q8_0, 32, 8, [260] * 130, F, H, True, False, {}),                          # CTA pairs, over 128 groups
    (Q6_K, 256, 392, [9, 100, 0, 17, 64, 65], H, H, True, True, {}),
    (Q5_K, 256, 2048, [1] * 20 + [40] * 3, H, F, False, True, {"tail": 2}),
    (Q8_0, 160, 136, [33, 64, 31], H, F, True, False, {"pad_x": 1})])
def test_grouped(samq, oracle, qtype, k, n, sizes, x_dtype, y_dtype, gelu, gather, extra):
    got, ref, tol = grouped_case(samq, oracle, qtype, k, n, sizes, x_dtype, y_dtype, gelu, gather, **extra)
    assert_close(got, ref, tol)
    samq.check(0)


@pytest.mark.parametrize("sizes", [[3, 2], [90, 100]])
def test_grouped_keeps_bad_rows_to_themselves(samq, oracle, sizes):
    """A row of NaN or infinities makes only its own outputs so."""
    def poison(x):
        x[1, 5] = np.nan
        x[4, :3] = np.inf
    got, ref, tol = grouped_case(samq, oracle, Q8_0, 96, 40, sizes, H, F, False, False, poison=poison)
    bad = [1, 4]
    assert not np.isfinite(got[bad]).any()
    good = np.setdiff1d(np.arange(sum(sizes)), bad)
    assert_close(got[good], ref[good], tol[good])


def test_grouped_reports_unusable_f32_activations(samq, oracle):
    rows, _ = packed(oracle, np.random.default_rng(0), Q8_0, 64, 64)
    w = samq.Weights(Q8_0, 64, 64, rows)
    x = torch.ones(4, 64, device="cuda")
    x[2, 3] = 7e4
    y = torch.empty(4, 32, device="cuda")
    samq.linear_grouped(w, 2, x, 4, 64, dev(np.array([0, 1, 4], np.int32)), 4, y, 32)
    with pytest.raises(samq.SamqError, match="SAMQ_ERR_RANGE"):
        samq.check(0)
    samq.check(0)
    w.close()


@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("indexed", [False, True])
def test_grouped_does_not_look_at_rows_outside_the_groups(samq, oracle, rows, indexed):
    """Unusable f32 values before and behind the plan (a padded batch) are neither read nor reported."""
    gguf, w64 = packed(oracle, np.random.default_rng(0), Q8_0, 2 * 32, 64)
    w = samq.Weights(Q8_0, 64, 64, gguf)
    x = torch.full((rows, 64), float("nan"), device="cuda")
    x[3:rows - 4] = torch.randn(rows - 7, 64, device="cuda")
    y = torch.full((rows, 32), SENTINEL, device="cuda")
    off = np.array([3, rows // 2, rows - 4], np.int32)
    index = dev(np.arange(rows, dtype=np.int32)) if indexed else None
    samq.linear_grouped(w, 2, x, rows, 64, dev(off), rows, y, 32, row_index=index)
    samq.check(0)
    xo = operand64(oracle, host(x)[3:rows - 4])
    got = host(y)
    assert (got[:3] == SENTINEL).all() and (got[rows - 4:] == SENTINEL).all()
    ref = np.stack([(w64[:32] if i + 3 < off[1] else w64[32:]) @ xo[i] for i in range(len(xo))])
    mag = np.stack([np.abs(w64[:32] if i + 3 < off[1] else w64[32:]) @ np.abs(xo[i]) for i in range(len(xo))])
    assert_close(got[3:rows - 4], ref, accumulation(64, mag) + 2.0 ** -24 * np.abs(ref))
    w.close()


@pytest.mark.parametrize("offsets", [[-5, 2, 99], [4, 1, 6], [0, 1 << 30, 3], [9, 9, 9]])
def test_grouped_bad_offsets_stay_inside(samq, oracle, offsets):
    """Offsets out of order or out of range write no row outside [0, rows)."""
    rows, _ = packed(oracle, np.random.default_rng(0), Q8_0, 64, 64)
    w = samq.Weights(Q8_0, 64, 64, rows)
    y = torch.full((10, 32), SENTINEL, device="cuda")
    samq.linear_grouped(w, 2, torch.ones(8, 64, device="cuda", dtype=torch.float16), 8, 64,
                        dev(np.array(offsets, np.int32)), 8, y, 32)
    assert (host(y)[8:] == SENTINEL).all()
    samq.check(0)
    w.close()


@pytest.mark.parametrize("rows,ld", [(70000, 32768), (5, (1 << 29) + 8)])
def test_grouped_offsets_beyond_32_bits(samq, oracle, rows, ld):
    """x and y of more than 2^31 elements: the last rows are right."""
    k, n = 32, 16
    gguf, w64 = packed(oracle, np.random.default_rng(1), Q8_0, 2 * n, k)
    w = samq.Weights(Q8_0, k, 2 * n, gguf)
    x = torch.empty(rows, ld, dtype=torch.float16, device="cuda")
    y = torch.empty(rows, ld, dtype=torch.float16, device="cuda")
    x[:, :k] = torch.randn(rows, k, device="cuda", dtype=torch.float16)
    y[:, :n] = SENTINEL
    cut = rows // 2
    samq.linear_grouped(w, 2, x, rows, ld, dev(np.array([0, cut, rows - 1], np.int32)), rows, y, ld)
    for r in (0, cut - 1, cut, rows - 2):
        wg = w64[:n] if r < cut else w64[n:]
        xr = host(x[r, :k]).astype(np.float64)
        ref, tol = finished(wg @ xr, accumulation(k, np.abs(wg) @ np.abs(xr)), False, H)
        assert_close(host(y[r, :n]), ref, tol, r)
    assert (host(y[rows - 1, :n]) == SENTINEL).all()
    w.close()
    del x, y
    torch.cuda.empty_cache()


def test_grouped_one_group_is_the_plain_linear(samq, oracle):
    """One group of all rows against samq_linear_f16_v1 on the same weights: the same operands and products."""
    rng = np.random.default_rng(11)
    rows, w64 = packed(oracle, rng, Q8_0, 264, 512)
    w = samq.Weights(Q8_0, 512, 264, rows)
    for m in (7, 150):
        x = rng.normal(0, 1, (m, 512)).astype(np.float16)
        a, b = (torch.empty(m, 264, device="cuda") for _ in range(2))
        samq.linear_f16(w, dev(x), m, 512, None, 0, a, 264)
        samq.linear_grouped(w, 1, dev(x), m, 512, dev(np.array([0, m], np.int32)), m, b, 264)
        tol = 2 * accumulation(512, np.abs(x.astype(np.float64)) @ np.abs(w64).T)
        assert_close(host(b), host(a).astype(np.float64), tol)
    w.close()


@pytest.mark.parametrize("qtype,k", [(Q8_0, 96), (Q8_0, 320), (Q4_K, 512), (Q5_K, 512), (Q6_K, 512)])
@pytest.mark.parametrize("n,groups", [(128, 2), (200, 3), (40, 7)])
def test_grouped_decodes_every_weight(samq, oracle, qtype, k, n, groups):
    """Unit vectors as activations read the weight operand back, bit for bit, whichever kernel multiplies."""
    rng = np.random.default_rng(k + n)
    gguf, w64 = packed(oracle, rng, qtype, groups * n, k)
    weights = samq.Weights(qtype, k, groups * n, gguf)
    for rows_each in (4, 100):
        rows = rows_each * groups
        for base in range(0, k, rows_each):
            cols = (base + np.arange(rows)) % k
            x = np.zeros((rows, k), H)
            x[np.arange(rows), cols] = 1
            y = torch.empty(rows, (n + 3) // 4 * 4, device="cuda")
            samq.linear_grouped(weights, groups, dev(x), rows, k, dev(np.arange(groups + 1, dtype=np.int32) * rows_each),
                                rows, y, y.shape[1])
            want = np.stack([w64[(i // rows_each) * n:(i // rows_each + 1) * n, cols[i]] for i in range(rows)])
            np.testing.assert_array_equal(host(y)[:, :n], want.astype(F))
    weights.close()


# ---- combine --------------------------------------------------------------------

@pytest.mark.parametrize("tokens,top_k,width,dtype,residual,in_place", [
    (1, 1, 8, H, False, False), (5, 3, 1000, H, True, False), (300, 8, 1024, F, True, True),
    (33, 32, 64, H, True, True), (2, 2, 4, F, False, False), (4000, 2, 256, H, True, False)])
def test_combine(samq, tokens, top_k, width, dtype, residual, in_place):
    rng = np.random.default_rng(tokens + width)
    y_rows = tokens * top_k
    unit = 8 if dtype == H else 4
    ldy, ldo = width + unit, width + 8
    y = np.full((y_rows, ldy), np.nan, dtype)
    y[:, :width] = rng.normal(0, 1, (y_rows, width))
    slots = rng.permutation(y_rows).astype(np.int32).reshape(tokens, top_k)
    weights = rng.random((tokens, top_k)).astype(np.float32)
    if tokens > 2:
        slots[0] = -1
        slots[1, 0] = y_rows
        weights[1, 0] = np.nan  # not read as a factor
        slots[2] = slots[2, 0]  # the same row several times
    res = rng.normal(0, 1, (tokens, ldo)).astype(np.float32) if residual else None
    out = torch.full((tokens, ldo), SENTINEL, device="cuda")
    if in_place:
        out.copy_(dev(res))
    rt = out if in_place else None if res is None else dev(res)
    samq.combine(dev(y), y_rows, ldy, dev(slots), dev(weights), tokens, top_k, width, out, ldo, residual=rt, ldr=ldo)
    got = host(out)
    ok = (slots >= 0) & (slots < y_rows)
    terms = np.where(ok[..., None], y[np.clip(slots, 0, y_rows - 1)][..., :width].astype(np.float64) *
                     np.where(ok, weights, 0).astype(np.float64)[..., None], 0)
    base = res[:, :width].astype(np.float64) if residual else np.zeros((tokens, width))
    tol = (top_k + 1) * 2.0 ** -24 * (np.abs(terms).sum(1) + np.abs(base))
    assert_close(got[:, :width], terms.sum(1) + base, tol + 2.0 ** -149)
    assert (got[:, width:] == (res[:, width:] if in_place else SENTINEL)).all()


# ---- adapters ---------------------------------------------------------------------

def adapters_case(samq, oracle, qtype, k, n, m, max_rank, count, x_dtype, y_dtype, gelu, ids=None, ranks=None,
                  bias=True, pad_x=0, pad_y=0, seed=0, poison=None):
    rng = np.random.default_rng(seed + m + 3 * n + k)
    gguf, w = packed(oracle, rng, qtype, n, k)
    unit_x, unit_y = (8 if x_dtype == H else 4), (8 if y_dtype == H else 4)
    ldx = k + pad_x * unit_x
    ldy = (n + unit_y - 1) // unit_y * unit_y + pad_y * unit_y
    x = np.full((m, ldx), 1e4, x_dtype)
    x[:, :k] = rng.normal(0, 1, (m, k))
    if poison is not None:
        poison(x)
    if ids is None:
        ids = rng.integers(-1, count, m)
    ids = np.asarray(ids, np.int32)
    b = rng.normal(0, 0.3, n).astype(np.float32) if bias else None
    weights = samq.Weights(qtype, k, n, gguf)
    ad = samq.Adapters(k, n, max_rank, count)
    ranks = ranks if ranks is not None else [max_rank] * count
    A, B, S = [], [], []
    for i in range(count):
        a = rng.normal(0, 1 / math.sqrt(k), (ranks[i], k)).astype(H)
        bb = rng.normal(0, 0.2, (n, ranks[i])).astype(H)
        s = float(np.float32(rng.uniform(0.5, 2)))
        if ranks[i]:
            if i % 2:
                ad.set(i, a.astype(F), bb.astype(F), s)
            else:
                ad.set(i, a, bb, s)
        A.append(a.astype(np.float64))
        B.append(bb.astype(np.float64))
        S.append(s)
    y = torch.full((m, ldy), SENTINEL, dtype=torch.float16 if y_dtype == H else torch.float32, device="cuda")
    space = samq.linear_adapters_workspace(weights, ad, m, torch.float16 if x_dtype == H else torch.float32)
    samq.linear_adapters(weights, ad, dev(x), m, ldx, dev(ids), y, ldy, bias=None if b is None else dev(b),
                         epilogue=1 if gelu else 0,
                         workspace=torch.full((space,), 255, dtype=torch.uint8, device="cuda"))
    got = host(y)
    ad.close()
    weights.close()
    xo = operand64(oracle, x[:, :k])
    with np.errstate(invalid="ignore"):
        pre = xo @ w.T + (b if bias else 0.0)
        tol = accumulation(k + 2 * max_rank, np.abs(xo) @ np.abs(w).T + (np.abs(b) if bias else 0.0))
        for i in range(count):
            mine = ids == i
            if not mine.any() or not ranks[i]:
                continue
            h = S[i] * (xo[mine] @ A[i].T)
            # the down product's accumulation, the scale's rounding, the f16 pair (2^-22, 2^-25 below normal)
            h_off = accumulation(k, S[i] * (np.abs(xo[mine]) @ np.abs(A[i]).T)) + 2.0 ** -22 * np.abs(h) + 2.0 ** -25
            pre[mine] += h @ B[i].T
            tol[mine] += h_off @ np.abs(B[i]).T + accumulation(k + 2 * max_rank, np.abs(h) @ np.abs(B[i]).T)
        ref, tol = finished(pre, tol, gelu, y_dtype)
    assert (got[:, n:] == SENTINEL).all(), "columns behind n changed"
    return got[:, :n], ref, tol


@pytest.mark.parametrize("qtype,k,n,m,rank,count,x_dtype,y_dtype,gelu,extra", [
    (Q8_0, 32, 8, 1, 1, 1, H, F, False, {"ids": [0]}),
    (Q8_0, 96, 201, 5, 3, 2, H, H, False, {"pad_x": 1, "pad_y": 1}),
    (Q4_K, 256, 384, 16, 16, 16, H, H, True, {"ids": list(range(16))}),
    (Q4_K, 1024, 136, 64, 17, 5, F, F, False, {}),
    (Q5_K, 512, 264, 65, 64, 3, H, F, True, {"bias": False}),
    (Q6_K, 768, 320, 130, 128, 4, F, H, False, {"pad_y": 1}),
    (Q8_0, 1056, 640, 257, 8, 40, H, H, False, {}),
    (Q8_0, 512, 200, 700, 33, 3, F, F, True, {"pad_x": 2}),
    (Q8_0, 256, 72, 300, 16, 300, H, F, False, {"ids": list(range(300))}),
    (Q8_0, 1024, 512, 1025, 64, 2, H, H, True, {"ids": [0] * 400 + [-1] * 225 + [1] * 400}),
    (Q8_0, 128, 64, 40, 16, 6, H, F, False, {"ranks": [0, 16, 5, 0, 1, 9]}),
    (Q8_0, 128, 136, 400, 48, 6, H, F, False, {"ranks": [0, 48, 5, 0, 1, 33]}),
    (Q8_0, 64, 40, 9, 4, 2, H, F, False, {"ids": [-1, 2, 1, -(1 << 31), 0, 1 << 30, 1, 0, -7]}),
    (Q8_0, 64, 40, 200, 4, 2, H, F, False, {"ids": [-1] * 200}),
    (Q4_K, 2048, 264, 256, 40, 80, H, F, False, {}),
    (Q8_0, 1024, 1032, 31, 100, 31, F, H, True, {"ids": list(range(31))})])
def test_adapters(samq, oracle, qtype, k, n, m, rank, count, x_dtype, y_dtype, gelu, extra):
    got, ref, tol = adapters_case(samq, oracle, qtype, k, n, m, rank, count, x_dtype, y_dtype, gelu, **extra)
    assert_close(got, ref, tol)
    samq.check(0)


@pytest.mark.parametrize("m", [6, 150])
def test_adapters_keep_bad_rows_to_themselves(samq, oracle, m):
    def poison(x):
        x[1, 5] = np.nan
        x[4, :3] = np.inf
    got, ref, tol = adapters_case(samq, oracle, Q8_0, 96, 40, m, 8, 3, H, F, False, poison=poison)
    bad = [1, 4]
    assert not np.isfinite(got[bad]).any()
    good = np.setdiff1d(np.arange(m), bad)
    assert_close(got[good], ref[good], tol[good])
    try:
        samq.check(0)
    except samq.SamqError as e:  # the bad rows' own finding, where their row has an adapter
        assert "SAMQ_ERR_RANGE" in str(e)
    samq.check(0)


@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("value,over", [(600.0, True), (400.0, False)])
def test_adapters_report_a_down_product_beyond_f16(samq, oracle, m, value, over):
    """128 x 600 = 76800 lies beyond the f16 operand range, 128 x 400 = 51200 within it."""
    k, n = 128, 64
    rows, _ = packed(oracle, np.random.default_rng(0), Q8_0, n, k)
    w = samq.Weights(Q8_0, k, n, rows)
    ad = samq.Adapters(k, n, 8, 1)
    ad.set(0, np.full((8, k), value, F), np.zeros((n, 8), F), 1.0)
    y = torch.empty(m, n, device="cuda")
    ids = np.full(m, -1, np.int32)
    ids[m // 2] = 0
    samq.linear_adapters(w, ad, torch.ones(m, k, dtype=torch.float16, device="cuda"), m, k, dev(ids), y, n)
    if over:
        with pytest.raises(samq.SamqError, match="SAMQ_ERR_RANGE"):
            samq.check(0)
    samq.check(0)
    ad.close()
    w.close()


def test_adapter_slots_change(samq, oracle):
    """A slot set again, cleared, or refused acts from the next call on."""
    rng = np.random.default_rng(3)
    k, n, m = 64, 40, 8
    rows, w64 = packed(oracle, rng, Q8_0, n, k)
    w = samq.Weights(Q8_0, k, n, rows)
    ad = samq.Adapters(k, n, 8, 2)
    x = rng.normal(0, 1, (m, k)).astype(H)
    ids = dev(np.full(m, 1, np.int32))
    y = torch.empty(m, n, device="cuda")
    base = x.astype(np.float64) @ w64.T
    mag = np.abs(x.astype(np.float64)) @ np.abs(w64).T

    def call():
        samq.linear_adapters(w, ad, dev(x), m, k, ids, y, n)
        return host(y).astype(np.float64)

    assert_close(call(), base, accumulation(k, mag) + 1e-30)
    for rank in (8, 3):
        a, b = rng.normal(0, 0.1, (rank, k)).astype(H), rng.normal(0, 0.1, (n, rank)).astype(H)
        ad.set(1, a, b, 2.0)
        delta = 2.0 * (x.astype(np.float64) @ a.astype(np.float64).T) @ b.astype(np.float64).T
        assert_close(call(), base + delta, 4 * accumulation(k + 16, mag + np.abs(x) @ np.abs(a.T) @ np.abs(b.T)) + 1e-6)
    before = call()
    bad = np.full((n, 3), 7e4, F)  # not finite in f16
    with pytest.raises(samq.SamqError, match="SAMQ_ERR_PAYLOAD"):
        ad.set(1, a.astype(F), bad, 1.0)
    with pytest.raises(samq.SamqError, match="SAMQ_ERR_PAYLOAD"):
        ad.set(1, a, b, float("nan"))
    np.testing.assert_array_equal(call(), before)
    ad.clear(1)
    assert_close(call(), base, accumulation(k, mag) + 1e-30)
    ad.close()
    w.close()


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [1, 37, 600])
def test_mixture_of_experts_layer(samq, oracle, tokens):
    """x + combine(fc2(gelu(fc1(x[rows])))) on the router's plan, on another stream, replayed from a graph."""
    rng = np.random.default_rng(tokens)
    E, K, MID, top_k = 6, 256, 512, 2
    g1, w1 = packed(oracle, rng, Q4_K, E * MID, K)
    g2, w2 = packed(oracle, rng, Q8_0, E * K, MID)
    h1, h2 = samq.Weights(Q4_K, K, E * MID, g1), samq.Weights(Q8_0, MID, E * K, g2)
    b1, b2 = rng.normal(0, 0.1, (E, MID)).astype(F), rng.normal(0, 0.1, (E, K)).astype(F)
    items = tokens * top_k
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = torch.empty(tokens, K, device="cuda")
        logits = torch.empty(tokens, E, device="cuda")
        weights, ids, offsets, rows, slots = torch.empty(tokens, top_k, device="cuda"), i32(tokens, top_k), \
            i32(E + 1), i32(items), i32(tokens, top_k)
        mid = torch.empty(items, MID, dtype=torch.float16, device="cuda")
        out, total = torch.empty(items, K, device="cuda"), torch.empty(tokens, K, device="cuda")
        tb1, tb2 = dev(b1), dev(b2)

        def layer():
            samq.route(logits, tokens, E, E, top_k, weights, ids, offsets, rows, slots)
            samq.linear_grouped(h1, E, x, tokens, K, offsets, items, mid, MID, row_index=rows, bias=tb1, epilogue=1)
            samq.linear_grouped(h2, E, mid, items, MID, offsets, items, out, K, bias=tb2)
            samq.combine(out, items, K, slots, weights, tokens, top_k, K, total, K, residual=x, ldr=K)

        def fill(seed):
            r = np.random.default_rng(seed)
            xv, lv = r.normal(0, 1, (tokens, K)).astype(F), r.normal(0, 1, (tokens, E)).astype(F)
            lv[0, :] = -np.inf  # a token without experts keeps its residual
            x.copy_(dev(xv))
            logits.copy_(dev(lv))
            return xv, lv

        def check(xv, lv):
            p, ident, off, rws, sl = route_reference(lv, top_k, True)
            xo = operand64(oracle, xv)
            ref = xv.astype(np.float64).copy()
            tol = 2.0 ** -22 * np.abs(ref)
            for t in range(tokens):
                for j in range(top_k):
                    e = ident[t, j]
                    if e < 0:
                        continue
                    a1, a2 = w1[e * MID:(e + 1) * MID], w2[e * K:(e + 1) * K]
                    pre = a1 @ xo[t] + b1[e]
                    hid, hid_off = finished(pre, accumulation(K, np.abs(a1) @ np.abs(xo[t]) + np.abs(b1[e])), True, H)
                    ref[t] += p[t, j] * (a2 @ hid + b2[e])
                    off2 = accumulation(MID, np.abs(a2) @ np.abs(hid) + np.abs(b2[e])) + np.abs(a2) @ hid_off
                    tol[t] += p[t, j] * off2 + 2.0 ** -20 * np.abs(p[t, j] * (a2 @ hid + b2[e]))
            assert_close(host(total), ref, tol)

        xv, lv = fill(1)
        layer()
        stream.synchronize()
        check(xv, lv)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer()
        for seed in (2, 3):
            xv, lv = fill(seed)
            graph.replay()
            stream.synchronize()
            check(xv, lv)
    samq.check(0)
    h1.close()
    h2.close()


FIRST_CALL_IN_A_GRAPH = """
import sys
sys.path[:0] = {paths!r}
import numpy as np
import torch
import samq
from oracle import oracle as o
samq.init(0)
rng = np.random.default_rng(0)
E, K, N, T, J = 4, 256, 128, {tokens}, 2
rows = o.quantize(o.Q8_0, rng.normal(0, 0.02, (E * N, K)).astype(np.float32))
w = samq.Weights(o.Q8_0, K, E * N, rows)
ad = samq.Adapters(K, N, 8, 2)
ad.set(0, rng.normal(0, 0.1, (8, K)).astype(np.float16), rng.normal(0, 0.1, (N, 8)).astype(np.float16), 1.0)
one = samq.Weights(o.Q8_0, K, N, rows.reshape(-1)[:N * o.row_bytes(o.Q8_0, K)])
x = torch.randn(T, K, device="cuda")
logits = torch.randn(T, E, device="cuda")
i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
weights, ids, off, plan, slots = torch.zeros(T, J, device="cuda"), i32(T, J), i32(E + 1), i32(T * J), i32(T, J)
y, out, z = torch.zeros(T * J, N, device="cuda"), torch.zeros(T, N, device="cuda"), torch.zeros(T, N, device="cuda")
who = i32(T)
def calls():
    samq.route(logits, T, E, E, J, weights, ids, off, plan, slots)
    samq.linear_grouped(w, E, x, T, K, off, T * J, y, N, row_index=plan)
    samq.combine(y, T * J, N, slots, weights, T, J, N, out, N)
    samq.linear_adapters(one, ad, x, T, K, who, z, N)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
graph.replay()
torch.cuda.synchronize()
first = [t.clone() for t in (weights, ids, off, plan, slots, y, out, z)]
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, (weights, ids, off, plan, slots, y, out, z)))
assert out.abs().sum() > 0 and z.abs().sum() > 0
samq.check(0)
print("same")
"""


@pytest.mark.parametrize("tokens", [5, 300])
def test_the_first_calls_may_be_captured(tokens):
    """In a fresh process, nothing but samq_init_v1 and the handles before the capture."""
    import subprocess
    import sys
    from conftest import PACKAGE, ROOT
    code = FIRST_CALL_IN_A_GRAPH.format(paths=[str(ROOT), str(PACKAGE)], tokens=tokens)
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]


def test_two_graphs_with_workspaces_of_their_own(samq, oracle):
    """Two captured calls of different sizes replayed on two streams at once."""
    rng = np.random.default_rng(9)
    k, n = 256, 136
    rows, w64 = packed(oracle, rng, Q8_0, n, k)
    w = samq.Weights(Q8_0, k, n, rows)
    ad = samq.Adapters(k, n, 16, 3)
    A, B = [], []
    for i in range(3):
        A.append(rng.normal(0, 0.05, (16, k)).astype(H))
        B.append(rng.normal(0, 0.2, (n, 16)).astype(H))
        ad.set(i, A[i], B[i], 1.0)
    jobs = []
    for m in (12, 500):
        x = rng.normal(0, 1, (m, k)).astype(F)
        ids = rng.integers(0, 3, m).astype(np.int32)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            job = {"x": dev(x), "ids": dev(ids), "y": torch.zeros(m, n, device="cuda"), "stream": s,
                   "space": torch.empty(samq.linear_adapters_workspace(w, ad, m, torch.float32), dtype=torch.uint8,
                                        device="cuda")}
            samq.linear_adapters(w, ad, job["x"], m, k, job["ids"], job["y"], n, workspace=job["space"])
            s.synchronize()
            job["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(job["graph"], stream=s):
                samq.linear_adapters(w, ad, job["x"], m, k, job["ids"], job["y"], n, workspace=job["space"])
            job["y"].zero_()
            s.synchronize()
        xo = operand64(oracle, x)
        h = np.stack([xo[i] @ A[ids[i]].astype(np.float64).T for i in range(m)])
        ref = xo @ w64.T + np.stack([h[i] @ B[ids[i]].astype(np.float64).T for i in range(m)])
        mag = np.abs(xo) @ np.abs(w64).T + np.stack(
            [np.abs(xo[i]) @ np.abs(A[ids[i]].astype(np.float64)).T @ np.abs(B[ids[i]].astype(np.float64)).T
             for i in range(m)])
        job["ref"], job["tol"] = ref, 3 * accumulation(k + 32, mag) + 1e-6
        jobs.append(job)
    for _ in range(20):
        for job in jobs:
            with torch.cuda.stream(job["stream"]):
                job["graph"].replay()
    torch.cuda.synchronize()
    for job in jobs:
        assert_close(host(job["y"]), job["ref"], job["tol"])
    samq.check(0)
    ad.close()
    w.close()


@pytest.mark.parametrize("as_address", [False, True])
def test_a_workspace_taken_by_the_call_belongs_to_its_stream(samq, oracle, as_address):
    """A call on another stream than the current one, without a workspace: what the current stream allocates and
    fills while the call has yet to run does not touch the call's memory."""
    rng = np.random.default_rng(12)
    k, n, m = 256, 128, 96
    rows, _ = packed(oracle, rng, Q8_0, n, k)
    w = samq.Weights(Q8_0, k, n, rows)
    x = dev(rng.normal(0, 1, (m, k)).astype(F))
    off = dev(np.array([0, m], np.int32))
    ref, y = torch.zeros(m, n, device="cuda"), torch.zeros(m, n, device="cuda")
    samq.linear_grouped(w, 1, x, m, k, off, m, ref, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # some 25 ms
    samq.linear_grouped(w, 1, x, m, k, off, m, y, n, stream=side.cuda_stream if as_address else side)
    size = samq.linear_grouped_workspace(w, 1, m, m, torch.float32, indexed=False)
    filled = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    del filled
    assert torch.equal(y, ref)
    samq.linear_grouped(w, 1, x, m, k, off, m, y.zero_(), n, stream=0)  # the default stream by its address
    assert torch.equal(y, ref)
    samq.check(0)
    w.close()


def test_calls_are_repeatable(samq, oracle):
    """The same call twice gives the same bits (no order of arrival decides a sum)."""
    for sizes in ([1, 3, 0, 2], [70, 3, 200, 1]):
        a = grouped_case(samq, oracle, Q4_K, 1024, 264, sizes, H, F, True, True)[0]
        b = grouped_case(samq, oracle, Q4_K, 1024, 264, sizes, H, F, True, True)[0]
        np.testing.assert_array_equal(a, b)
    for m in (20, 300):
        a = adapters_case(samq, oracle, Q4_K, 1024, 264, m, 16, 5, H, F, False)[0]
        b = adapters_case(samq, oracle, Q4_K, 1024, 264, m, 16, 5, H, F, False)[0]
        np.testing.assert_array_equal(a, b)


# ---- several units of work a CTA -------------------------------------------------------
# The packet kernel's CTAs are one an SM; beyond 148 weight row tiles (groups x n / 128) each works through several, so
# that its rings of copies wrap around from one to the next.

@pytest.mark.parametrize("qtype,k,n,m,rank,count,x_dtype,y_dtype,gelu,extra", [
    (Q4_K, 1024, 19072, 16, 16, 16, H, F, False, {"ids": list(range(16))}),
    (Q8_0, 1024, 40000, 64, 16, 40, H, H, False, {}),
    (Q5_K, 512, 28680, 31, 128, 12, H, F, False, {}),
    (Q6_K, 768, 19200, 64, 128, 10, F, F, False, {}),
    (Q4_K, 256, 32000, 33, 8, 33, H, F, False, {"ids": list(range(33))}),
    (Q8_0, 96, 40008, 9, 4, 9, F, H, False, {"ids": list(range(9))}),
    (Q6_K, 1024, 19072, 5, 16, 3, H, F, False, {"bias": False}),
    (Q5_K, 512, 19072, 32, 16, 32, H, F, True, {"ids": list(range(32))})])
def test_adapters_of_wide_projections(samq, oracle, qtype, k, n, m, rank, count, x_dtype, y_dtype, gelu, extra):
    got, ref, tol = adapters_case(samq, oracle, qtype, k, n, m, rank, count, x_dtype, y_dtype, gelu, **extra)
    assert_close(got, ref, tol)
    again = adapters_case(samq, oracle, qtype, k, n, m, rank, count, x_dtype, y_dtype, gelu, **extra)[0]
    np.testing.assert_array_equal(got, again)
    samq.check(0)


@pytest.mark.parametrize("qtype,k,n,sizes,x_dtype", [
    (Q8_0, 1024, 2504, [9, 16, 1, 7] * 4, H), (Q6_K, 1024, 2504, [16, 1, 0, 12] * 5, F),     # 16 rows at a time
    (Q4_K, 1024, 2504, [20, 32, 17] * 4, H), (Q5_K, 512, 2504, [32, 30, 29] * 4, F),         # 32
    (Q6_K, 2048, 2504, [18, 25, 32] * 4, H), (Q8_0, 1056, 2504, [31, 17, 26] * 4, F),
    (Q8_0, 1024, 2504, [64, 40, 50, 33] * 3, H), (Q4_K, 1024, 2504, [60, 35, 64, 50] * 3, F),  # 64
    (Q5_K, 2048, 2504, [64, 64, 33, 48] * 3, H), (Q6_K, 1024, 2504, [36, 64, 41, 64] * 3, F),
    (Q8_0, 1024, 40008, [64], H), (Q5_K, 512, 40008, [33], F), (Q4_K, 256, 40008, [1], H)])
def test_grouped_of_many_units(samq, oracle, qtype, k, n, sizes, x_dtype):
    got, ref, tol = grouped_case(samq, oracle, qtype, k, n, sizes, x_dtype, F, False, False)
    assert_close(got, ref, tol)
    for _ in range(2):
        again = grouped_case(samq, oracle, qtype, k, n, sizes, x_dtype, F, False, False)[0]
        np.testing.assert_array_equal(got, again)
    samq.check(0)


@pytest.mark.parametrize("m", [9, 400])
@pytest.mark.parametrize("scale", [1.0, 0.1, 1e-3, 1e-5, 1e-7, 2.0 ** -27, 3000.0])
def test_adapters_keep_the_down_product_to_the_stated_bound(samq, oracle, m, scale):
    """Through a zero W and a B of ones the output is h = scale A x itself: within 2^-22 |h| + 2^-25 of it (the f16
    pair), and the f32 arithmetic beside that: one rounding by the scale, truncated sums of two terms."""
    rng = np.random.default_rng(int(m + 1e9 * scale))
    k, r = 64, 16
    w = samq.Weights(Q8_0, k, r, oracle.quantize(Q8_0, np.zeros((r, k), F)))
    ad = samq.Adapters(k, r, r, 1)
    a = np.zeros((r, k), H)
    a[np.arange(r), rng.permutation(k)[:r]] = rng.uniform(0.5, 2, r).astype(H)  # one product of 22 bits each: exact
    ad.set(0, a, np.eye(r, dtype=H), scale)
    x = (rng.uniform(0.5, 4, (m, k)) * rng.choice([-1, 1], (m, k))).astype(H)
    y = torch.empty(m, r, device="cuda")
    samq.linear_adapters(w, ad, dev(x), m, k, dev(np.zeros(m, np.int32)), y, r)
    samq.check(0)
    h = float(np.float32(scale)) * (x.astype(np.float64) @ a.astype(np.float64).T)
    off = np.abs(host(y) - h)
    assert (off <= (2.0 ** -22 + 2.0 ** -24 + 2.0 ** -23) * np.abs(h) + 2.0 ** -25).all(), float((off / np.abs(h)).max())
    ad.close()
    w.close()


def test_binding_refuses_what_the_sizes_do_not_fit(samq, oracle):
    """Tensors that are too small, not contiguous, or strided otherwise than stated are refused before any launch; views
    whose rows lie the stated stride apart are taken."""
    t, e, j, k, n = 70, 4, 2, 64, 32
    logits = torch.randn(t, e + 2, device="cuda")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    route = {"logits": logits[:, 1:e + 1], "tokens": t, "experts": e, "ld": e + 2, "top_k": j,
             "weights": torch.zeros(t, j, device="cuda"), "ids": i32(t, j), "offsets": i32(e + 1), "rows": i32(t * j),
             "slots": i32(t, j)}
    samq.route(**route)
    for name, bad in (("ids", i32(j, t).t()), ("slots", i32(t - 1, j)), ("offsets", i32(e)), ("rows", i32(t * j, 2)[:, 0]),
                      ("weights", torch.zeros(t, 2 * j, device="cuda")[:, :j]), ("logits", logits[:, 3:]),
                      ("logits", logits[1:]), ("logits", logits.t())):
        with pytest.raises(ValueError):
            samq.route(**{**route, name: bad})
    rows, _ = packed(oracle, np.random.default_rng(0), Q8_0, e * n, k)
    w, one = samq.Weights(Q8_0, k, e * n, rows), samq.Weights(Q8_0, k, n, rows.reshape(-1)[:rows.size // e])
    x = torch.randn(t, k + 8, device="cuda", dtype=torch.float16)
    y = torch.zeros(t * j, n + 8, device="cuda")
    grouped = {"w": w, "groups": e, "x": x[:, 8:], "x_rows": t, "ldx": k + 8, "offsets": route["offsets"], "rows": t * j,
               "y": y[:, 4:], "ldy": n + 8, "row_index": route["rows"], "bias": torch.zeros(e, n, device="cuda")}
    samq.linear_grouped(**grouped)
    for name, bad in (("x", x[1:]), ("x", x[:, 16:]), ("y", y[:, 12:]), ("offsets", i32(e)), ("row_index", i32(t)),
                      ("bias", torch.zeros(n, device="cuda")), ("rows", t * j + 1), ("x_rows", t + 1), ("ldx", k),
                      ("workspace", torch.zeros(8, dtype=torch.uint8, device="cuda").expand(1 << 16, 8))):
        with pytest.raises(ValueError):
            samq.linear_grouped(**{**grouped, name: bad})
    combine = {"y": y[:, 4:], "y_rows": t * j, "ldy": n + 8, "slots": route["slots"], "weights": route["weights"],
               "tokens": t, "top_k": j, "width": n, "out": torch.zeros(t, n, device="cuda"), "ldo": n,
               "residual": torch.zeros(t, n + 4, device="cuda")[:, :n], "ldr": n + 4}
    samq.combine(**combine)
    for name, bad in (("y_rows", t * j + 1), ("slots", i32(j, t).t()), ("weights", torch.zeros(t, device="cuda")),
                      ("out", torch.zeros(t - 1, n, device="cuda")), ("ldr", n), ("tokens", t + 1)):
        with pytest.raises(ValueError):
            samq.combine(**{**combine, name: bad})
    ad = samq.Adapters(k, n, 4, 2)
    adapters = {"w": one, "adapters": ad, "x": x[:, 8:], "m": t, "ldx": k + 8, "ids": i32(t), "y": y[:, 4:],
                "ldy": n + 8, "bias": torch.zeros(n, device="cuda")}
    samq.linear_adapters(**adapters)
    for name, bad in (("x", x[1:]), ("ids", i32(t - 1)), ("ids", i32(t, 2)[:, 1]), ("y", y[:t - 1]),
                      ("bias", torch.zeros(n - 1, device="cuda")), ("ldx", k), ("m", 2 * t + 1)):
        with pytest.raises(ValueError):
            samq.linear_adapters(**{**adapters, name: bad})
    samq.check(0)
    ad.close()
    w.close()
    one.close()

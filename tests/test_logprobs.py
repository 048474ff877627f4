"""lssm_logprobs / lssm_logprobs_backward (and the engine's scoring calls) against plain
implementations in 64 bits, at the sizes, types, strides and masks where they can go wrong.

Tolerances, derived from the arithmetic (u = 2^-24, the rounding of fp32):
  * s = sum e^d over V terms: a thread adds at most V / 256 + 1 of them in a row and the threads'
    sums are joined in about ten more additions; e^d itself is good to 2^-21 (d rounded once, times
    log2 e rounded once, an exponential of 2 ulp). So log s is within E = (V / 256 + 64) u absolutely,
    and u / s = sum p d within E (1 + sum p |d|).
  * lse = m + log s, logp = (x_t - m) - log s: E plus one rounding of each operand and result.
  * outputs of 16 bits: half a step (finfo.eps / 2) of the value.
"""

import numpy as np
import pytest

import lssm

U = 2.0 ** -24
NONE = lssm.NO_TOKEN


# ---- CPU: refusals, before any device is looked at ---------------------------------------------

def refuse(name, args, match):
    with pytest.raises(lssm.LssmError, match=match):
        lssm.check(getattr(lssm.lib(), name)(None, *args))


A = 0x10000  # an aligned address nothing dereferences: the calls are refused


@pytest.mark.parametrize("args,match", [
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 3, 0)), "dtype"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 0, 0, 0, 0)), "vocab must be"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 1 << 31, 4, 0, 0)), "vocab must be"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(1 << 31, 10, 4, 0, 0)), "rows must be"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 100, 33, 0, 0)), "top_k"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 11, 0, 0)), "top_k"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 9)), "row_stride"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 1 << 41)), "row_stride"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(1 << 20, 10, 4, 0, 1 << 40)), "row_stride"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 0, 0, 0)), "top_ids"),
    ((A, A, A, A, A, None, A, lssm.LogprobsDims(2, 10, 4, 0, 0)), "top_ids"),
    ((A, A, A, A, A, A, None, lssm.LogprobsDims(2, 10, 4, 0, 0)), "top_ids"),
    ((A, A, None, None, None, None, None, lssm.LogprobsDims(2, 10, 0, 0, 0)), "no output"),
    ((None, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 0)), "null logits"),
    ((A, None, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 0)), "logp needs targets"),
    ((A + 1, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 0)), "aligned"),
    ((A + 2, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 2, 0)), "aligned"),
    ((A, A + 2, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 0)), "aligned"),
    ((A, A, A, A, A, A, A, lssm.LogprobsDims(2, 10, 4, 0, 0)), "null context"),
])
def test_logprobs_refuses(args, match):
    refuse("lssm_logprobs", args, match)


@pytest.mark.parametrize("args,match", [
    ((A, A, A, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 3, 0, 0, 0)), "dtype"),
    ((A, A, A, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 3, 0, 0)), "dtype"),
    ((A, A, A, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 0, 0, 0, 0, 0)), "vocab"),
    ((A, A, A, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 0, 9, 0)), "row_stride"),
    ((A, A, A, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 9)), "grad_stride"),
    ((A, A, A, A, None, None, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "no gradient"),
    ((A, A, None, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "null"),
    ((A, A, A, A, A, A, None, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "null"),
    ((A, None, A, A, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "needs targets"),
    ((A, A, A, None, A, A, 2 * A, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "needs entropy"),
    ((A, A, A, A, A, A, 2 * A + 1, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "aligned"),
    ((A, A, A, A, A, A, A + 2, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "overlaps"),
    ((A, A, A, A, A, A, A, lssm.LogprobsGradDims(2, 10, 0, 2, 0, 0)), "overlaps"),
    ((A, A, A, A, A, A, A, lssm.LogprobsGradDims(2, 10, 0, 0, 12, 10)), "overlaps"),
    ((A, A, A, A, A, A, A, lssm.LogprobsGradDims(2, 10, 0, 0, 0, 0)), "null context"),
])
def test_logprobs_backward_refuses(args, match):
    refuse("lssm_logprobs_backward", args, match)


# ---- the definition in 64 bits -----------------------------------------------------------------

def bf16_bits(x):
    b = np.asarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def encode(x, dt):
    """(the array to upload, its values in 64 bits)"""
    x = np.asarray(x, np.float32)
    if dt == lssm.DT_F32:
        return x, x.astype(np.float64)
    with np.errstate(over="ignore"):
        if dt == lssm.DT_F16:
            return x.astype(np.float16), x.astype(np.float16).astype(np.float64)
    nan = np.isnan(x)
    b = bf16_bits(np.where(nan, 0, x))
    b[nan] = 0x7FC0
    return b, bf16_value(b).astype(np.float64)


def truth(x, t, k):
    """lse, logp, entropy, top ids and values of one row, from the definition."""
    n = len(x)
    ids = np.lexsort((np.arange(n), -np.where(np.isnan(x), -np.inf, x)))[:k].astype(np.uint32)
    if np.isnan(x).any() or np.isposinf(x).any():
        return np.nan, 0.0 if t == NONE else np.nan, np.nan, ids, np.full(k, np.nan)
    if np.isneginf(x).all():
        return -np.inf, 0.0 if t == NONE else np.nan if t >= n else -np.inf, 0.0, ids, np.full(k, -np.inf)
    m = x.max()
    e = np.exp(x - m)
    s = e.sum()
    lse = m + np.log(s)
    live = e > 0
    H = np.log(s) - (e[live] * (x[live] - m)).sum() / s
    logp = 0.0 if t == NONE else np.nan if t >= n else (x[t] - m) - np.log(s)
    return lse, logp, H, ids, (x[ids] - m) - np.log(s)


def within(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (got, want)
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)])
    ok = np.abs(got[~odd] - want[~odd]) <= np.broadcast_to(tol, got.shape)[~odd]
    assert ok.all(), (got[~odd][~ok][:4], want[~odd][~ok][:4], np.abs(got[~odd] - want[~odd])[~ok].max())


def call(ctx, arr, t, V, k, dt, stride=0, off=0, parts=("logp", "entropy", "lse")):
    """Runs lssm_logprobs over the uploaded `arr` (from element `off` on)."""
    rows = len(t)
    buf = lssm.DeviceBuffer.from_array(ctx, arr)
    bt = lssm.DeviceBuffer.from_array(ctx, np.asarray(t, np.uint32))
    out = {n: lssm.DeviceBuffer.from_array(ctx, np.full(rows + 1, 7.5, np.float32)) for n in parts}
    bi = lssm.DeviceBuffer.from_array(ctx, np.full(rows * k + 1, 77, np.uint32)) if k else None
    bv = lssm.DeviceBuffer.from_array(ctx, np.full(rows * k + 1, 7.5, np.float32)) if k else None
    x = lssm.DeviceView(ctx, buf.ptr.value + off * arr.itemsize)
    lssm.Ops(ctx).logprobs(x, bt, out.get("logp"), out.get("entropy"), out.get("lse"), bi, bv,
                           lssm.LogprobsDims(rows, V, k, dt, stride))
    got = {n: b.download(np.float32, rows + 1) for n, b in out.items()}
    assert all(v[rows] == 7.5 for v in got.values())
    got = {n: v[:rows] for n, v in got.items()}
    if k:
        ids, top = bi.download(np.uint32, rows * k + 1), bv.download(np.float32, rows * k + 1)
        assert ids[-1] == 77 and top[-1] == 7.5
        got["ids"], got["top"] = ids[:-1].reshape(rows, k), top[:-1].reshape(rows, k)
    return got


def check_rows(got, x64, t, V, k):
    E = (V / 256 + 64) * U
    for r in range(len(t)):
        lse, logp, H, ids, top = truth(x64[r], int(t[r]), k)
        big = max(abs(lse) if np.isfinite(lse) else 0.0, abs(logp) if np.isfinite(logp) else 0.0)
        spread = 1 + abs(H if np.isfinite(H) else 0.0) + (abs(lse - np.nanmax(x64[r])) if np.isfinite(lse) else 0.0)
        if "lse" in got:
            within(got["lse"][r], lse, E + 2 * U * big)
        if "logp" in got:
            within(got["logp"][r], logp, E + 2 * U * big)
        if "entropy" in got:
            within(got["entropy"][r], H, E * spread)
        if k:
            assert np.array_equal(got["ids"][r], ids), r
            within(got["top"][r], top, E + 2 * U * np.where(np.isfinite(top), np.abs(top), 0) + 2 * U * big)


def logits(rng, rows, V):
    x = rng.standard_normal((rows, V)) * 2.5
    x[np.arange(rows), rng.integers(0, V, rows)] += 8.0
    return x


DTYPES = [lssm.DT_F16, lssm.DT_BF16, lssm.DT_F32]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 33, 32), (4, 257, 7), (1, 4099, 20), (7, 9001, 32),
                                      (2, 50288, 20), (1, 65537, 5), (300, 515, 3), (1, 256000, 32), (64, 12345, 0)])
def test_logprobs(ctx, dt, rows, V, k):
    rng = np.random.default_rng(rows * 1000 + V + dt)
    arr, x64 = encode(logits(rng, rows, V), dt)
    t = rng.integers(0, V, rows).astype(np.uint32)
    t[rng.random(rows) < 0.2] = NONE
    check_rows(call(ctx, arr, t, V, k, dt), x64, t, V, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("pad,off", [(1, 0), (3, 1), (0, 1), (8, 5), (7, 3)])
def test_logprobs_strides_and_offsets(ctx, dt, pad, off):
    """Rows that start at every alignment; NaN between the rows is not read into them."""
    rows, V, k = 9, 1501, 6
    rng = np.random.default_rng(pad * 10 + off)
    full = np.full(off + rows * (V + pad), np.nan)
    x = logits(rng, rows, V)
    for r in range(rows):
        full[off + r * (V + pad):off + r * (V + pad) + V] = x[r]
    arr, _ = encode(full, dt)
    _, x64 = encode(x, dt)
    t = rng.integers(0, V, rows).astype(np.uint32)
    check_rows(call(ctx, arr, t, V, k, dt, stride=V + pad, off=off), x64, t, V, k)


def odd_rows(dt, V, rng):
    """Rows that masks and ties leave: (values, target)."""
    lowest = {lssm.DT_F16: -65504.0, lssm.DT_BF16: -3.3895e38, lssm.DT_F32: -3.4028234e38}[dt]
    inf, x = np.inf, logits(rng, 1, V)[0]
    one = np.full(V, -inf); one[V // 2] = 1.5
    last = np.full(V, -inf); last[V - 1] = -3.0
    few = np.where(rng.random(V) < 0.97, -inf, x)
    few[0] = 0.25
    low = np.where(rng.random(V) < 0.9, lowest, x)
    nan = x.copy(); nan[V // 3] = np.nan
    pinf = x.copy(); pinf[V // 3] = inf
    both = few.copy(); both[1] = np.nan
    zeros = np.zeros(V); zeros[::2] = -0.0
    up, down = np.linspace(-20, 20, V), np.linspace(20, -20, V)
    two = np.full(V, lowest); two[3] = lowest / 2
    return [(np.full(V, -inf), 0), (np.full(V, -inf), NONE), (np.full(V, -inf), V + 5), (one, V // 2), (one, 0), (last, V - 1), (few, 0),
            (low, 1), (np.full(V, lowest), 2), (two, 3), (nan, 0), (nan, NONE), (pinf, V // 3), (both, 0), (zeros, 5), (np.full(V, 3.0), V - 1),
            (up, 0), (down, 0), (x, NONE), (x, V), (x, NONE - 1), (np.full(V, 60000.0) + x, 4), (x * 1000, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,k", [(40, 32), (1003, 20), (30011, 32)])
def test_logprobs_masks_ties_and_non_finite(ctx, dt, V, k):
    rng = np.random.default_rng(V)
    rows = odd_rows(dt, V, rng)
    with np.errstate(over="ignore"):
        arr, x64 = encode(np.stack([r[0] for r in rows]), dt)
    t = np.array([r[1] for r in rows], np.uint32)
    check_rows(call(ctx, arr, t, V, k, dt), x64, t, V, k)


@pytest.mark.gpu
def test_logprobs_any_output_alone(ctx):
    rng = np.random.default_rng(3)
    arr, x64 = encode(logits(rng, 4, 777), lssm.DT_F16)
    t = rng.integers(0, 777, 4).astype(np.uint32)
    whole = call(ctx, arr, t, 777, 5, lssm.DT_F16)
    for parts, k in ((("logp",), 0), (("entropy",), 0), (("lse",), 0), ((), 5), (("logp", "lse"), 5)):
        got = call(ctx, arr, t, 777, k, lssm.DT_F16, parts=parts)
        for n in parts:
            np.testing.assert_allclose(got[n], whole[n], rtol=0, atol=(777 / 256 + 64) * U * 8)
        if k:
            assert np.array_equal(got["ids"], whole["ids"])
    b = lssm.DeviceBuffer.from_array(ctx, arr)
    e = lssm.DeviceBuffer(ctx, 16)
    lssm.Ops(ctx).logprobs(b, None, None, e, None, None, None, lssm.LogprobsDims(4, 777, 0, lssm.DT_F16, 0))   # no targets
    np.testing.assert_allclose(e.download(np.float32, 4), whole["entropy"], rtol=0, atol=1e-4)
    lssm.Ops(ctx).logprobs(None, None, e, None, None, None, None, lssm.LogprobsDims(0, 777, 0, lssm.DT_F16, 0))   # no rows
    lssm.Ops(ctx).logprobs(None, None, e, None, None, None, None, lssm.LogprobsDims(0, 777, 0, lssm.DT_F16, 0))


def grad_truth(x, t, g, h):
    if np.isneginf(x).all():
        return np.zeros(len(x))
    lse, _, H, _, _ = truth(x, NONE, 0)
    lp = x - lse
    p = np.exp(lp)
    d = np.zeros(len(x))
    if t != NONE:
        d -= g * p
        d[t] += g
    live = p > 0
    d[live] -= h * p[live] * (lp[live] + H)
    return d


def backward(ctx, arr, t, lse, ent, g, h, V, dt, gdt, stride=0, gstride=0, in_place=False):
    rows = len(t)
    f = lambda a: None if a is None else lssm.DeviceBuffer.from_array(ctx, np.asarray(a, np.float32))  # noqa: E731
    buf = lssm.DeviceBuffer.from_array(ctx, arr)
    np_t = {lssm.DT_F16: np.float16, lssm.DT_BF16: np.uint16, lssm.DT_F32: np.float32}[gdt]
    n = rows * (gstride or V)
    out = buf if in_place else lssm.DeviceBuffer.from_array(ctx, np.full(n + 1, 3, np_t))
    lssm.Ops(ctx).logprobs_backward(buf, lssm.DeviceBuffer.from_array(ctx, np.asarray(t, np.uint32)), f(lse), f(ent), f(g), f(h), out,
                                    lssm.LogprobsGradDims(rows, V, dt, gdt, stride, gstride))
    got = out.download(np_t, n if in_place else n + 1)
    if not in_place:
        assert got[n] == 3
        between = got[:n].reshape(rows, gstride or V)[:, V:]
        assert (between == 3).all()
    got = got[:n].reshape(rows, gstride or V)[:, :V]
    return bf16_value(got).astype(np.float64) if gdt == lssm.DT_BF16 else got.astype(np.float64)


HALF_STEP = {lssm.DT_F16: 2.0 ** -11, lssm.DT_BF16: 2.0 ** -8, lssm.DT_F32: U}


def check_grad(got, x64, t, g, h, gdt):
    """p is off by the roundings of lse (given in fp32), of x - lse and of the exponential."""
    for r in range(len(t)):
        want = grad_truth(x64[r], int(t[r]), g[r], h[r])
        lse, _, H, _, _ = truth(x64[r], NONE, 0)
        if not np.isfinite(lse):
            assert np.array_equal(got[r], want)
            continue
        lp = x64[r] - lse
        p = np.exp(lp)
        lp = np.where(p > 0, lp, 0.0)
        rel = (4 * abs(lse) + 4 * np.abs(lp) + 16) * U
        size = (abs(g[r]) + abs(h[r]) * (np.abs(lp + H) + 1)) * p
        tol = HALF_STEP[gdt] * np.abs(want) + size * rel * (1 + HALF_STEP[gdt]) + abs(g[r]) * 2 * U * (np.arange(len(lp)) == t[r])
        tol += 2.0 ** -25 if gdt == lssm.DT_F16 else 2.0 ** -126
        bad = ~(np.abs(got[r] - want) <= tol)
        assert not bad.any(), (r, got[r][bad][:4], want[bad][:4], tol[bad][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("dt,gdt", [(a, b) for a in DTYPES for b in DTYPES])
@pytest.mark.parametrize("rows,V,pad,gpad", [(1, 1, 0, 0), (3, 37, 1, 0), (2, 1000, 0, 3), (5, 4099, 5, 5), (1, 50288, 0, 0)])
def test_logprobs_backward(ctx, dt, gdt, rows, V, pad, gpad):
    rng = np.random.default_rng(V + 7 * dt + gdt)
    full = np.full((rows, V + pad), np.nan)
    full[:, :V] = logits(rng, rows, V)
    arr, x64 = encode(full, dt)
    x64 = x64[:, :V]
    t = rng.integers(0, V, rows).astype(np.uint32)
    if rows > 2:
        t[1] = NONE
    g = np.float32(rng.standard_normal(rows) * 4)
    h = np.float32(rng.standard_normal(rows))
    tr = [truth(x, NONE, 0) for x in x64]
    lse, ent = [a[0] for a in tr], [a[2] for a in tr]
    for gg, hh in ((g, h), (g, None), (None, h)):
        got = backward(ctx, arr, t, lse, ent, gg, hh, V, dt, gdt, V + pad, V + gpad)
        check_grad(got, x64, t if gg is not None else np.full(rows, NONE, np.uint32), gg if gg is not None else 0 * g,
                   hh if hh is not None else 0 * h, gdt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_logprobs_backward_in_place(ctx, dt):
    rng = np.random.default_rng(11)
    arr, x64 = encode(logits(rng, 3, 2053), dt)
    t = np.array([5, NONE, 2052], np.uint32)
    tr = [truth(x, NONE, 0) for x in x64]
    g, h = np.float32([2, 3, -1]), np.float32([0.5, -1, 1])
    got = backward(ctx, arr, t, [a[0] for a in tr], [a[2] for a in tr], g, h, 2053, dt, dt, in_place=True)
    check_grad(got, x64, t, g, h, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_logprobs_backward_masks(ctx, dt):
    """Forward outputs fed back: masked entries and empty rows give zeros, what is NaN stays NaN."""
    V = 203
    rows = [r for r in odd_rows(dt, V, np.random.default_rng(5)) if r[1] == NONE or r[1] < V]
    with np.errstate(over="ignore"):
        arr, x64 = encode(np.stack([r[0] for r in rows]), dt)
    t = np.array([r[1] for r in rows], np.uint32)
    f = call(ctx, arr, t, V, 0, dt)
    g, h = np.full(len(t), 2.0, np.float32), np.full(len(t), 0.5, np.float32)
    got = backward(ctx, arr, t, f["lse"], f["entropy"], g, h, V, dt, lssm.DT_F32)
    sick = np.isnan(f["lse"])
    assert np.isnan(got[sick]).all()
    ok = np.flatnonzero(~sick)
    # lse here is the forward kernel's: its own tolerance adds to p's
    E = (V / 256 + 64) * U
    for r in ok:
        want = grad_truth(x64[r], int(t[r]), 2.0, 0.5)
        lse = truth(x64[r], NONE, 0)[0]
        big = abs(lse) if np.isfinite(lse) else 0.0
        tol = (np.abs(want) + 2.5 * (1 + np.log(V))) * (E + 8 * U * big) + 2 * U
        assert (np.abs(got[r] - want) <= tol).all(), (r, np.abs(got[r] - want).max())
    bad = backward(ctx, arr[:1] if arr.ndim == 1 else np.ascontiguousarray(arr[-1:]), [V], [f["lse"][-1]], [f["entropy"][-1]], [1.0], None, V, dt,
                   lssm.DT_F32)
    assert np.isnan(bad).all()   # a target outside the vocabulary


@pytest.mark.gpu
def test_logprobs_gradient_against_differences(ctx):
    """d/dx of sum_r (g logp + h entropy) by central differences of the 64-bit forward."""
    V = 23
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, V)).astype(np.float32)
    t, g, h = np.array([4, 22], np.uint32), np.float32([1.5, -2]), np.float32([0.7, 1.1])
    tr = [truth(r.astype(np.float64), NONE, 0) for r in x]
    got = backward(ctx, x, t, [a[0] for a in tr], [a[2] for a in tr], g, h, V, lssm.DT_F32, lssm.DT_F32)

    def total(z):
        a = [truth(z[r], int(t[r]), 0) for r in range(2)]
        return sum(g[r] * a[r][1] + h[r] * a[r][2] for r in range(2))

    d, z = 1e-5, x.astype(np.float64)
    for r in range(2):
        for j in range(V):
            up, dn = z.copy(), z.copy()
            up[r, j] += d
            dn[r, j] -= d
            # the differences' own error: d^2 / 6 times a third derivative of order 1, and 1e-16 / d
            assert abs((total(up) - total(dn)) / (2 * d) - got[r, j]) < 1e-8 + 64 * U


@pytest.mark.gpu
@pytest.mark.parametrize("V,k,rows", [(5003, 8, 3), (150001, 20, 2)])   # a CTA a row; a cluster a row
def test_logprobs_captured_and_replayed(ctx, V, k, rows):
    """The call in a captured batch, replayed on new logits in the same buffers."""
    rng = np.random.default_rng(2)
    c = lssm.Ctx(0)
    c.set_graph_batching(True)
    b = lssm.DeviceBuffer.from_array(c, encode(logits(rng, rows, V), lssm.DT_F16)[0])
    t = rng.integers(0, V, rows).astype(np.uint32)
    bt = lssm.DeviceBuffer.from_array(c, t)
    o = [lssm.DeviceBuffer(c, rows * 4) for _ in range(3)]
    bi, bv = lssm.DeviceBuffer(c, rows * k * 4), lssm.DeviceBuffer(c, rows * k * 4)
    c.begin_batch()
    lssm.Ops(c).logprobs(b, bt, *o, bi, bv, lssm.LogprobsDims(rows, V, k, lssm.DT_F16, 0))
    c.commit_and_wait()
    for _ in range(2):
        arr, x64 = encode(logits(rng, rows, V), lssm.DT_F16)
        b.upload(arr)
        c.replay_batch(1)
        got = dict(zip(("logp", "entropy", "lse"), (q.download(np.float32, rows) for q in o)))
        got["ids"], got["top"] = bi.download(np.uint32, rows * k).reshape(rows, k), bv.download(np.float32, rows * k).reshape(rows, k)
        check_rows(got, x64, t, V, k)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,k,rows", [(64003, 32, 3), (128000, 7, 2), (256001, 20, 5)])
def test_logprobs_in_clusters(ctx, dt, V, k, rows):
    """Rows split over 2, 4 and 8 CTAs: equal entries, masks and the largest entry in every slice."""
    rng = np.random.default_rng(V)
    x = np.round(logits(rng, rows, V), 1)          # many equal entries
    x[0, V // 2:] = -np.inf                        # a slice, or half of them, with nothing left
    x[1] = np.where(rng.random(V) < 0.9999, -np.inf, x[1])
    x[rows - 1, [0, V // 3, V - 1]] = 30.0
    arr, x64 = encode(x, dt)
    t = np.array([V - 1, 5, V // 3, 0, NONE][:rows], np.uint32)
    check_rows(call(ctx, arr, t, V, k, dt), x64, t, V, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,pad,off,k", [(1, 0, 0, 1), (5, 2, 3, 2), (1501, 6, 1, 4), (12007, 1, 0, 3)])
def test_logprobs_more_rows_than_ctas(ctx, dt, V, pad, off, k):
    """Rows of later waves, whose beginnings earlier ones ask for: the last rows end with the array."""
    rows = 1400
    rng = np.random.default_rng(V)
    few = np.pad(logits(rng, 35, V), ((0, 0), (0, pad)))
    full = np.concatenate([np.zeros(off), np.tile(few, (rows // 35, 1)).ravel()])[:off + rows * (V + pad) - pad]
    arr, _ = encode(full, dt)
    _, x64 = encode(few[:, :V], dt)
    t = rng.integers(0, V, rows).astype(np.uint32)
    check_rows(call(ctx, arr, t, V, k, dt, stride=V + pad, off=off), np.tile(x64, (rows // 35, 1)), t, V, k)


@pytest.mark.gpu
def test_logprobs_two_contexts_on_streams_of_their_own(ctx):
    """Calls of two contexts in flight together do not meet: nothing is shared between them."""
    rng = np.random.default_rng(4)
    V, k, rows = 40009, 9, 40
    cs = [lssm.Ctx(0), lssm.Ctx(0)]
    made = []
    for c in cs:
        arr, x64 = encode(logits(rng, rows, V), lssm.DT_F16)
        t = rng.integers(0, V, rows).astype(np.uint32)
        bufs = [lssm.DeviceBuffer.from_array(c, arr), lssm.DeviceBuffer.from_array(c, t)]
        out = [lssm.DeviceBuffer(c, rows * 4) for _ in range(3)] + [lssm.DeviceBuffer(c, rows * k * 4) for _ in range(2)]
        made.append((x64, t, bufs, out))
    for c in cs:
        c.begin_batch()
    for _ in range(20):
        for c, (x64, t, bufs, out) in zip(cs, made):
            lssm.Ops(c).logprobs(*bufs, *out, lssm.LogprobsDims(rows, V, k, lssm.DT_F16, 0))
    for c in cs:
        c.commit_and_wait()
    for x64, t, bufs, out in made:
        got = dict(zip(("logp", "entropy", "lse"), (q.download(np.float32, rows) for q in out)))
        got["ids"], got["top"] = out[3].download(np.uint32, rows * k).reshape(rows, k), out[4].download(np.float32, rows * k).reshape(rows, k)
        check_rows(got, x64, t, V, k)
    for c in cs:
        c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_logprobs_backward_target_outside_the_vocabulary(ctx, dt):
    """Such a row is NaN throughout: masked entries, entries whose p is 0 and rows that a mask leaves empty among them,
    with either gradient or both. Rows beside it are not touched by it."""
    V = 203
    rng = np.random.default_rng(7)
    x = logits(rng, 6, V)
    x[1, ::3] = -np.inf
    x[2] = -np.inf
    x[3, 1:] -= 2000.0
    arr, x64 = encode(x, dt)
    t = np.array([V, V + 1, V, NONE - 1, 3, NONE], np.uint32)
    tr = [truth(r, NONE, 0) for r in x64]
    lse, ent = [a[0] for a in tr], [a[2] for a in tr]
    g, h = np.full(6, 1.5, np.float32), np.full(6, -0.5, np.float32)
    for gg, hh in ((g, None), (g, h), (None, h)):
        got = backward(ctx, arr, t, lse, ent, gg, hh, V, dt, lssm.DT_F32)
        assert np.isnan(got[:4]).all()
        check_grad(got[4:], x64[4:], t[4:] if gg is not None else np.full(2, NONE, np.uint32), (gg if gg is not None else 0 * g)[4:],
                   (hh if hh is not None else 0 * h)[4:], lssm.DT_F32)

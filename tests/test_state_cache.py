"""The quantised state cache (lssm_state_cache_*, lssm_ssd_step_cached) against a plain
implementation in 64 bits: the recurrence token by token over the codes as they stand.

Tolerances, derived from the arithmetic (u = 2^-24):
  * codes of a stored state: the scale is one correctly rounded division and the code the nearest
    whole number to the exact quotient, so codes and scales equal the reference's bit for bit;
  * S and y before rounding: W + 1 products and sums for an element, N more for y (in lanes): below 64 u
    of the sum of the terms' sizes. A term that was decayed by exp(-e) is off by 12 e u more: e is a sum
    of products of a rate (an exponential, 4 u) and dt (log1p of an exponential, 6 u), each rounded,
    and what e is off by absolutely the term is off by relatively. `err` carries that part;
  * y is rounded to fp16: half a step, 2^-11; a loaded state to its type's half step;
  * a folded state is within half a step of its codes, scale / 2, of S.
"""

import numpy as np
import pytest

import lssm

U = 2.0 ** -24
DT_MIN, DT_MAX = 1e-6, 1e6


# ---- CPU ------------------------------------------------------------------------------------------

def dims(batch=2, H=4, P=8, N=16, G=1, window=4, bits=8, has_D=1):
    return lssm.StateCacheDims(batch, H, P, N, G, window, bits, DT_MIN, DT_MAX, has_D)


BAD = [(dict(bits=4), "bits must be 8 or 16"), (dict(bits=0), "bits"), (dict(window=0), "window"), (dict(window=33), "window"),
       (dict(H=5, G=2), "multiple of n_groups"), (dict(batch=1 << 20, H=1 << 12), "too large"), (dict(P=1 << 17), "too large"),
       (dict(N=1 << 17), "too large")]


def cache_ptrs(**kw):
    c = dict(codes=0x1000, scales=0x2000, win_x=0x3000, win_B=0x4000, win_dt=0x5000, fill=0x6000)
    c.update(kw)
    return lssm.StateCachePtrs(*(c[n] for n in ("codes", "scales", "win_x", "win_B", "win_dt", "fill")))


def store_args(d, c, state=0x10000):
    return "lssm_state_cache_store", (state, c, d)


def load_args(d, c, A=0x8000, state=0x10000, dt=2):
    return "lssm_state_cache_load", (c, A, state, dt, d)


def step_args(d, c, **kw):
    a = dict(x=0x100, B=0x200, C=0x300, dt=0x400, bias=0x500, A=0x600, D=0x700, y=0x800)
    a.update(kw)
    return "lssm_ssd_step_cached", (a["x"], a["B"], a["C"], a["dt"], a["bias"], a["A"], a["D"], c, a["y"], d)


def refuse(call, match):
    name, args = call
    with pytest.raises(lssm.LssmError, match=match):
        lssm.check(getattr(lssm.lib(), name)(None, *args))


@pytest.mark.parametrize("kw,match", BAD)
def test_shapes_refused(kw, match):
    d, c = dims(**kw), cache_ptrs()
    for call in (store_args(d, c), load_args(d, c), step_args(d, c)):
        refuse(call, match)
    with pytest.raises(lssm.LssmError, match=match):
        lssm.check(lssm.lib().lssm_state_cache_bytes(d, (lssm.u64 * 6)()))


@pytest.mark.parametrize("which", ["codes", "scales", "win_x", "win_B", "win_dt", "fill"])
def test_null_and_misaligned_arrays_refused(which):
    d = dims(bits=16)
    for make in (store_args, load_args, step_args):
        refuse(make(d, cache_ptrs(**{which: None})), "null cache array")
        refuse(make(d, cache_ptrs(**{which: 0x1001})), "not aligned")


@pytest.mark.parametrize("which", ["x", "B", "C", "dt", "bias", "A", "D", "y"])
def test_step_arguments_refused(which):
    refuse(step_args(dims(), cache_ptrs(), **{which: None}), "null array")
    refuse(step_args(dims(), cache_ptrs(), **{which: 0x101}), "not aligned")


def test_load_and_store_arguments_refused():
    d, c = dims(), cache_ptrs()
    refuse(store_args(d, c, None), "null or misaligned state")
    refuse(store_args(d, c, 0x10002), "null or misaligned state")
    refuse(load_args(d, c, A=None), "null or misaligned")
    refuse(load_args(d, c, state=None), "null or misaligned")
    refuse(load_args(d, c, state=0x10002), "null or misaligned")
    refuse(load_args(d, c, dt=3), "dtype")
    refuse(store_args(d, c), "null context")
    refuse(load_args(d, c), "null context")
    refuse(step_args(d, c), "null context")
    refuse(step_args(dims(has_D=0), c, D=None), "null context")   # D is not looked at without has_D
    nothing = cache_ptrs(**{n: None for n in ("codes", "scales", "win_x", "win_B", "win_dt", "fill")})
    for kw in (dict(batch=0), dict(H=0), dict(P=0), dict(N=0)):   # an empty cache has no arrays
        for call in (store_args(dims(**kw), nothing, None), load_args(dims(**kw), nothing, None, None), step_args(dims(**kw), nothing)):
            refuse(call, "null context")


def test_bytes():
    n = (lssm.u64 * 6)()
    lssm.check(lssm.lib().lssm_state_cache_bytes(dims(3, 6, 5, 7, 2, 9, 16), n))
    assert list(n) == [3 * 6 * 5 * 7 * 2, 3 * 6 * 5 * 4, 3 * 9 * 6 * 5 * 2, 3 * 9 * 2 * 7 * 2, 3 * 6 * 9 * 4, 3 * 6 * 4]
    lssm.check(lssm.lib().lssm_state_cache_bytes(dims(64, 128, 128, 65535, 8, 32, 16), n))
    assert n[0] == 64 * 128 * 128 * 65535 * 2   # beyond 32 bits


# ---- the definition -------------------------------------------------------------------------------

def quantise(S, bits):
    """(codes, fp32 scales) of states (.., N) in 64 bits."""
    Q = 127 if bits == 8 else 32767
    S = np.asarray(S, np.float64)
    amax = np.abs(S).max(-1)
    with np.errstate(over="ignore", invalid="ignore"):
        scale = (amax / Q).astype(np.float32)
        scale[scale < np.finfo(np.float32).tiny] = 0
        scale[~np.isfinite(amax)] = np.nan
        s = scale.astype(np.float64)[..., None]
        code = np.where(s > 0, np.rint(S / np.where(s > 0, s, 1)), 0)
    return np.clip(code, -Q, Q).astype(np.int8 if bits == 8 else np.int16), scale


class Cache:
    """A cache on the device and the same in 64 bits, fed with the same tokens."""

    def __init__(self, ctx, d, rng, S=None):
        self.ctx, self.d, self.ops = ctx, d, lssm.Ops(ctx)
        self.B, self.H, self.P, self.N = d.batch, d.H, d.P, d.N
        self.G = d.n_groups or 1
        self.cache = lssm.StateCache(ctx, d)
        self.A_log = np.log(rng.uniform(1, 16, self.H)).astype(np.float16)
        self.bias = (rng.standard_normal(self.H) * 0.7 - 3.5).astype(np.float16)
        self.D = rng.uniform(0, 1, self.H).astype(np.float16)
        up = lambda a: lssm.DeviceBuffer.from_array(ctx, a)  # noqa: E731
        self.dA, self.dbias, self.dD = up(self.A_log), up(self.bias), up(self.D)
        shape = (self.B, self.H, self.P, self.N)
        if S is None:
            S = rng.standard_normal(shape) * np.exp(rng.standard_normal((*shape[:3], 1)))
        self.S0 = np.asarray(S, np.float32)
        self.dS = up(self.S0)
        self.ops.state_cache_store(self.dS, self.cache, d)
        self.pull()

    def codes(self):
        n = self.B * self.H * self.P * self.N
        return self.cache.buffers[0].download(np.int8 if self.d.bits == 8 else np.int16, n).reshape(self.B, self.H, self.P, self.N)

    def scales(self):
        return self.cache.buffers[1].download(np.float32, self.B * self.H * self.P).reshape(self.B, self.H, self.P)

    def fill(self):
        return self.cache.buffers[5].download(np.uint32, self.B * self.H).reshape(self.B, self.H)

    def pull(self):
        """The reference's state becomes what the device's codes stand for."""
        with np.errstate(invalid="ignore"):
            self.S = self.codes().astype(np.float64) * self.scales().astype(np.float64)[..., None]
        self.size = np.abs(self.S)   # the sizes of the terms an element was summed from
        self.err = np.zeros_like(self.size)   # what their decays are off by

    def token(self, rng):
        B, H, P, N, G = self.B, self.H, self.P, self.N, self.G
        r = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
        return r(B, H, P), r(B, G, N), r(B, G, N), (rng.standard_normal((B, H)) * 0.7).astype(np.float16)

    def advance(self, tok):
        """The recurrence in 64 bits; returns y before its rounding and how far it may be off."""
        x, Bm, Cm, raw = (a.astype(np.float64) for a in tok)
        v = (tok[3].astype(np.float32) + self.bias.astype(np.float32)).astype(np.float64)
        dt = np.clip(np.where(v > 20, v, np.log1p(np.exp(np.minimum(v, 30)))), np.float64(np.float32(DT_MIN)), np.float64(np.float32(DT_MAX)))
        a = -np.exp(self.A_log.astype(np.float64))
        per = self.H // self.G
        Bh, Ch = np.repeat(Bm, per, 1), np.repeat(Cm, per, 1)
        decay = np.exp(a * dt)[..., None, None]
        add = (dt[..., None] * x)[..., None] * Bh[:, :, None, :]
        self.S = decay * self.S + add
        e = np.minimum(-a * dt, 700)[..., None, None]
        self.err = decay * (self.err + 12 * U * e * self.size) + 12 * U * np.abs(add)
        self.size = decay * self.size + np.abs(add)
        D = self.D.astype(np.float64)[None, :, None] if self.d.has_D else 0.0
        y = (self.S * Ch[:, :, None, :]).sum(-1) + D * x
        size = (self.size * np.abs(Ch)[:, :, None, :]).sum(-1) + np.abs(D * x)
        return y, 64 * U * size + (self.err * np.abs(Ch)[:, :, None, :]).sum(-1)

    def tol(self):
        return 64 * U * self.size + self.err

    def step(self, tok, ctx=None):
        ops = lssm.Ops(ctx) if ctx else self.ops
        up = lambda a: lssm.DeviceBuffer.from_array(self.ctx, a)  # noqa: E731
        n = self.B * self.H * self.P
        y = up(np.full(n + 1, 9, np.float16))
        ops.ssd_step_cached(*(up(a) for a in tok), self.dbias, self.dA, self.dD if self.d.has_D else None, self.cache, y, self.d)
        got = y.download(np.float16, n + 1)
        assert got[n] == 9
        return got[:n].reshape(self.B, self.H, self.P).astype(np.float64)

    def load(self, dt=lssm.DT_F32):
        n = self.S.size
        t = {lssm.DT_F16: np.float16, lssm.DT_BF16: np.uint16, lssm.DT_F32: np.float32}[dt]
        out = lssm.DeviceBuffer.from_array(self.ctx, np.full(n + 1, 5, t))
        self.ops.state_cache_load(self.cache, self.dA, out, dt, self.d)
        got = out.download(t, n + 1)
        assert got[n] == 5
        got = got[:n]
        if dt == lssm.DT_BF16:
            got = (got.astype(np.uint32) << 16).view(np.float32)
        return got.astype(np.float64).reshape(self.S.shape)


def run_tokens(c, rng, tokens, check_every=1):
    Q = 127 if c.d.bits == 8 else 32767
    fill = int(c.fill()[0, 0])
    for i in range(tokens):
        tok = c.token(rng)
        got = c.step(tok)
        y, off_y = c.advance(tok)
        tol = 2.0 ** -11 * np.abs(y) + off_y + 2.0 ** -25
        bad = ~(np.abs(got - y) <= tol)
        assert not bad.any(), (i, got[bad][:4], y[bad][:4], tol[bad][:4])
        fill += 1
        if fill == c.d.window:
            fill = 0
            scale = c.scales().astype(np.float64)
            amax = np.abs(c.S).max(-1)
            assert (np.abs(scale - amax / Q) <= (c.tol().max(-1) + U * amax) / Q + 1e-38).all()
            held = c.codes().astype(np.float64) * scale[..., None]
            off = np.abs(held - c.S)
            lim = scale[..., None] / 2 * (1 + 2.0 ** -20) + c.tol() + c.tol().max(-1, keepdims=True)
            assert (off <= lim).all(), (off - lim).max()
            c.pull()
        assert (c.fill() == fill).all()
        if i % check_every == 0:
            assert (np.abs(c.load() - c.S) <= c.tol() + U * np.abs(c.S)).all()


# (batch, H, P, N, G, window): the common shape; odd and tiny ones; several groups; W = 1 and 32
SHAPES = [(3, 4, 64, 128, 1, 16), (1, 24, 64, 128, 1, 16), (2, 8, 64, 128, 4, 5), (2, 3, 64, 128, 1, 32), (1, 2, 64, 128, 1, 1),
          (2, 2, 16, 128, 2, 17), (1, 1, 1, 1, 1, 1), (2, 6, 5, 7, 3, 3), (1, 3, 48, 75, 1, 8), (2, 2, 33, 300, 1, 4), (1, 5, 128, 256, 5, 16),
          (2, 4, 80, 128, 2, 12), (1, 3, 64, 64, 1, 16), (65, 2, 64, 128, 1, 4),
          # the other state sizes with whole rows, long windows; rows padded to 64, 128 and 256 columns; the most
          # shared memory; more rows or columns than the padded kernel holds
          (2, 4, 64, 64, 2, 21), (3, 3, 128, 256, 1, 32), (40, 8, 16, 64, 1, 3), (2, 3, 75, 203, 1, 16), (2, 2, 31, 100, 1, 30),
          (1, 2, 255, 255, 1, 20), (1, 1, 256, 256, 1, 5), (1, 2, 300, 40, 1, 3), (1, 2, 20, 260, 2, 18), (1, 1, 257, 261, 1, 32),
          (2, 1, 4, 36, 1, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("shape", SHAPES)
def test_steps_match_the_recurrence(ctx, shape, bits):
    B, H, P, N, G, W = shape
    rng = np.random.default_rng(B * 100 + N + bits)
    c = Cache(ctx, dims(B, H, P, N, G, W, bits), rng)
    codes, scales = quantise(c.S0, bits)
    assert np.array_equal(c.scales(), scales) and np.array_equal(c.codes(), codes)
    run_tokens(c, rng, min(2 * W + 1, 40), check_every=3)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
def test_without_D_and_groups_zero(ctx, bits):
    rng = np.random.default_rng(4)
    run_tokens(Cache(ctx, dims(2, 4, 64, 128, 0, 6, bits, has_D=0), rng), rng, 13)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,N", [(8, 128), (16, 128), (8, 33), (16, 33)])
def test_store_borders(ctx, bits, N):
    """Zero rows, tiny and huge rows, exact half steps, NaN and infinities, one element only."""
    Q = 127 if bits == 8 else 32767
    S = np.zeros((1, 1, 16, N), np.float32)
    r = np.random.default_rng(0).standard_normal(N).astype(np.float32)
    S[0, 0, 1] = r * 1e-44
    S[0, 0, 2] = r * 1e-38
    S[0, 0, 3] = r * 3e37
    S[0, 0, 4] = (np.arange(N) % (2 * Q)) + 0.5
    S[0, 0, 4, 0] = -Q                                    # scale 1: every half is a tie
    S[0, 0, 4] = np.clip(S[0, 0, 4], -Q, Q)
    S[0, 0, 5] = r; S[0, 0, 5, N - 1] = np.nan
    S[0, 0, 6] = r; S[0, 0, 6, 0] = np.inf
    S[0, 0, 7] = r; S[0, 0, 7, N // 2] = -np.inf
    S[0, 0, 8, N - 1] = -3.25
    S[0, 0, 9] = r * np.float32(1.17549435e-38 * Q)
    S[0, 0, 10] = -0.0
    S[0, 0, 11] = r * 1e30
    S[0, 0, 12] = np.nextafter(np.float32(0.5), np.float32(0)); S[0, 0, 12, 0] = Q
    S[0, 0, 13] = np.nextafter(np.float32(0.5), np.float32(1)); S[0, 0, 13, 0] = Q
    S[0, 0, 14:] = np.random.default_rng(1).standard_normal((2, N))
    rng = np.random.default_rng(3)
    c = Cache(ctx, dims(1, 1, 16, N, 1, 4, bits), rng, S)
    codes, scales = quantise(S, bits)
    assert np.array_equal(c.scales(), scales, equal_nan=True)
    assert np.array_equal(c.codes(), codes)
    got = c.load()
    assert np.isnan(got[0, 0, 5:8]).all() and (got[0, 0, [0, 1, 10]] == 0).all()
    fine = np.isfinite(S).all(-1)[0, 0]
    with np.errstate(invalid="ignore"):
        want = (codes.astype(np.float64) * scales.astype(np.float64)[..., None]).astype(np.float32)
    assert np.array_equal(got[0, 0, fine], want[0, 0, fine])


@pytest.mark.gpu
def test_store_many_random_rows_exact(ctx):
    """Codes next to half steps: 2 M elements, equal to the 64-bit rounding."""
    rng = np.random.default_rng(8)
    for bits, N in ((8, 128), (16, 128), (16, 77)):
        S = (rng.standard_normal((1, 128, 128, N)) * np.exp(rng.standard_normal((1, 128, 128, 1)) * 5)).astype(np.float32)
        c = Cache(ctx, dims(1, 128, 128, N, 1, 4, bits), rng, S)
        codes, scales = quantise(S, bits)
        assert np.array_equal(c.scales(), scales) and np.array_equal(c.codes(), codes)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 4, 64, 128, 1, 16), (1, 2, 7, 19, 2, 5), (1, 2, 255, 255, 1, 20), (2, 3, 75, 203, 1, 16),
                                   (1, 1, 256, 256, 1, 32), (2, 4, 48, 64, 2, 7), (1, 2, 33, 300, 1, 4), (3, 2, 40, 100, 1, 9)])
@pytest.mark.parametrize("dt,half", [(lssm.DT_F16, 2.0 ** -11), (lssm.DT_BF16, 2.0 ** -8), (lssm.DT_F32, U)])
def test_load_types(ctx, shape, dt, half):
    rng = np.random.default_rng(6)
    for bits in (8, 16):
        c = Cache(ctx, dims(*shape, bits), rng)
        tokens = 0
        for n in (0, 1, 3):
            for _ in range(n):
                tok = c.token(rng)
                c.step(tok)
                c.advance(tok)
                tokens += 1
                if tokens == shape[5]:   # folded: the state is what the codes hold (a window of 4 fills here)
                    c.pull()
            before = [b.download(np.uint8, b.nbytes) for b in c.cache.buffers]
            got = c.load(dt)
            assert (np.abs(got - c.S) <= half * np.abs(c.S) + c.tol() * (1 + half) + 2.0 ** -25).all()
            after = [b.download(np.uint8, b.nbytes) for b in c.cache.buffers]
            assert all(np.array_equal(x, y) for x, y in zip(before, after))   # a load changes nothing


@pytest.mark.gpu
@pytest.mark.parametrize("P,N", [(64, 128), (5, 9)])
def test_sequences_with_their_own_fill(ctx, P, N):
    """A sequence re-stored between steps (its arrays from its first element on) starts an empty
    window while the others go on; the batch steps them together."""
    rng = np.random.default_rng(12)
    H, G, W, B = 4, 2, 5, 3
    c = Cache(ctx, dims(B, H, P, N, G, W, 8), rng)
    one = dims(1, H, P, N, G, W, 8)
    sizes = (lssm.u64 * 6)()
    lssm.check(lssm.lib().lssm_state_cache_bytes(one, sizes))
    for i in range(2 * W + 2):
        if i == 3:
            part = lssm.StateCache.wrap(*(b.ptr.value + 1 * int(k) for b, k in zip(c.cache.buffers, sizes)))
            S = rng.standard_normal((1, H, P, N)).astype(np.float32)
            c.ops.state_cache_store(lssm.DeviceBuffer.from_array(ctx, S), part, one)
            codes, scales = quantise(S, 8)
            c.S[1] = codes[0].astype(np.float64) * scales[0].astype(np.float64)[..., None]
            c.size[1], c.err[1] = np.abs(c.S[1]), 0
        tok = c.token(rng)
        got = c.step(tok)
        y, off_y = c.advance(tok)
        assert (np.abs(got - y) <= 2.0 ** -11 * np.abs(y) + off_y + 2.0 ** -25).all()
        f = c.fill()
        assert (f == f[:, :1]).all()
        for b in range(B):
            assert f[b, 0] == ((i + 1) % W if b != 1 or i < 3 else (i - 2) % W)
            if f[b, 0] == 0:
                held = c.codes()[b].astype(np.float64) * c.scales()[b].astype(np.float64)[..., None]
                assert (np.abs(held - c.S[b]) <= c.scales()[b].astype(np.float64)[..., None] * (0.5 + 1e-4) + 2 * c.tol()[b].max()).all()
                c.S[b], c.size[b], c.err[b] = held, np.abs(held), 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
def test_extreme_steps(ctx, bits):
    """dt at both clamps, a decay that forgets everything, the largest x, and what is not finite."""
    rng = np.random.default_rng(2)
    c = Cache(ctx, dims(1, 4, 64, 128, 1, 6, bits), rng)
    for i in range(14):
        x, Bm, Cm, raw = c.token(rng)
        raw[0, 0] = -30.0          # dt clamped up to 1e-6
        raw[0, 1] = 300.0 if i % 4 == 1 else raw[0, 1]   # exp(a dt) = 0: only this token and later ones are left
        x[0, 2] = 60000.0 * np.sign(x[0, 2].astype(np.float32)).astype(np.float16)
        Cm = (Cm.astype(np.float32) * 1e-2).astype(np.float16)
        got = c.step((x, Bm, Cm, raw))
        y, off_y = c.advance((x, Bm, Cm, raw))
        tol = 2.0 ** -11 * np.abs(y) + off_y + 2.0 ** -25
        over = np.abs(y) > 65504
        assert (np.abs(got - y) <= tol)[~over].all()
        if (c.fill() == 0).all():
            c.pull()
    x, Bm, Cm, raw = c.token(rng)
    x[0, 3, 5] = np.nan
    got = c.step((x, Bm, Cm, raw))
    y, _ = c.advance((x, Bm, Cm, raw))
    assert np.array_equal(np.isnan(got), np.isnan(y)) and np.isnan(got).sum() == 1
    for _ in range(6):
        tok = c.token(rng)
        c.step(tok)
        c.advance(tok)
    got = c.load()
    assert np.isnan(got[0, 3, 5]).all() and np.isfinite(np.delete(got[0, 3], 5, 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
def test_captured_step_replays_through_a_fold(ctx, bits):
    """One captured step, replayed: the fill count lives on the device, so the fold comes on time."""
    rng = np.random.default_rng(9)
    cc = lssm.Ctx(0)
    c = Cache(cc, dims(2, 8, 64, 128, 1, 3, bits), rng)
    up = lambda a: lssm.DeviceBuffer.from_array(cc, a)  # noqa: E731
    tok = c.token(rng)
    bufs = [up(a) for a in tok]
    n = c.B * c.H * c.P
    y = lssm.DeviceBuffer(cc, n * 2)
    cc.set_graph_batching(True)
    cc.begin_batch()
    c.ops.ssd_step_cached(*bufs, c.dbias, c.dA, c.dD, c.cache, y, c.d)
    cc.commit_and_wait()
    cc.set_graph_batching(False)
    for i in range(8):
        if i:
            tok = c.token(rng)
            for b, a in zip(bufs, tok):
                b.upload(a)
            cc.replay_batch(1)
        got = y.download(np.float16, n).reshape(c.B, c.H, c.P).astype(np.float64)
        want, off_y = c.advance(tok)
        assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + off_y + 2.0 ** -25).all()
        if (c.fill() == 0).all():
            c.pull()
    cc.close()


@pytest.mark.gpu
def test_empty_calls_do_nothing(ctx):
    none = lssm.StateCache.wrap(None, None, None, None, None, None)
    ops = lssm.Ops(ctx)
    for kw in (dict(batch=0), dict(H=0), dict(P=0), dict(N=0)):
        d = dims(**kw)
        ops.state_cache_store(None, none, d)
        ops.state_cache_load(none, None, None, lssm.DT_F32, d)
        ops.ssd_step_cached(None, None, None, None, None, None, None, none, None, d)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 3, 64, 128, 1, 4), (1, 3, 75, 203, 1, 4), (2, 2, 17, 50, 1, 4)])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_load_to_16_bits_writes_nothing_else(ctx, shape, off):
    """A 16-bit state that begins at any element, with neighbours on both sides that stay as they are."""
    rng = np.random.default_rng(off)
    c = Cache(ctx, dims(*shape, 8), rng)
    tok = c.token(rng)
    c.step(tok)
    c.advance(tok)
    n = c.S.size
    buf = lssm.DeviceBuffer.from_array(ctx, np.full(n + off + 40, 7.5, np.float16))
    c.ops.state_cache_load(c.cache, c.dA, lssm.DeviceView(ctx, buf.ptr.value + 2 * off), lssm.DT_F16, c.d)
    got = buf.download(np.float16, n + off + 40)
    assert (got[:off] == 7.5).all() and (got[off + n:] == 7.5).all()
    held = got[off:off + n].reshape(c.S.shape).astype(np.float64)
    half = 2.0 ** -11
    assert (np.abs(held - c.S) <= half * np.abs(c.S) + c.tol() * (1 + half) + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("which", ["codes", "win_x", "win_B", "x", "B", "C", "state"])
def test_arrays_off_by_an_element(ctx, which, bits):
    """Arrays aligned to their element only: the common shape leaves its 16-byte path."""
    rng = np.random.default_rng(21)
    d = dims(2, 4, 64, 128, 1, 3, bits)
    c = Cache(ctx, d, rng)
    es = bits // 8 if which == "codes" else 4 if which == "state" else 2
    keep = []

    def shifted(a):
        raw = np.ascontiguousarray(a).view(np.uint8).reshape(-1)
        b = lssm.DeviceBuffer.from_array(ctx, np.concatenate([np.zeros(es, np.uint8), raw, np.zeros(64, np.uint8)]))
        keep.append(b)
        return lssm.DeviceView(ctx, b.ptr.value + es)

    names = ("codes", "scales", "win_x", "win_B", "win_dt", "fill")
    ptrs = dict(zip(names, (b.ptr.value for b in c.cache.buffers)))
    if which in ptrs:
        b = c.cache.buffers[names.index(which)]
        ptrs[which] = shifted(b.download(np.uint8, b.nbytes)).ptr.value
    cache = lssm.StateCache.wrap(*(ptrs[n] for n in names))
    up = lambda a, n: shifted(a) if n == which else lssm.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    for i in range(5):
        tok = c.token(rng)
        y = lssm.DeviceBuffer(ctx, c.B * c.H * c.P * 2)
        c.ops.ssd_step_cached(*(up(a, n) for a, n in zip(tok, ("x", "B", "C", "dt"))), c.dbias, c.dA, c.dD, cache, y, d)
        want, off_y = c.advance(tok)
        got = y.download(np.float16, c.B * c.H * c.P).reshape(c.B, c.H, c.P).astype(np.float64)
        assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + off_y + 2.0 ** -25).all()
        out = shifted(np.zeros(c.S.shape, np.float32)) if which == "state" else lssm.DeviceBuffer(ctx, c.S.size * 4)
        c.ops.state_cache_load(cache, c.dA, out, lssm.DT_F32, d)
        host = np.empty(c.S.size, np.float32)
        lssm.check(lssm.lib().lssm_download(ctx.h, host.ctypes.data_as(lssm.P), out.ptr, 0, host.nbytes))
        held = host.astype(np.float64).reshape(c.S.shape)
        if (i + 1) % 3 == 0:   # folded: within half a step of the state, and exactly what goes on from here
            Q = 127 if bits == 8 else 32767
            lim = np.abs(c.S).max(-1, keepdims=True) / Q * (0.5 + 1e-4) + 2 * c.tol().max(-1, keepdims=True)
            assert (np.abs(held - c.S) <= lim).all()
            c.S, c.size, c.err = held, np.abs(held), np.zeros_like(held)
        else:
            assert (np.abs(held - c.S) <= c.tol() + U * np.abs(c.S)).all()


class SizedTokens(Cache):
    """Tokens whose x, or whose B, differ in size by up to 2^30 from row to row, or from token to token."""

    def __init__(self, ctx, d, rng, kind, big):
        self.kind, self.big, self.made = kind, big, 0
        super().__init__(ctx, d, rng, np.zeros((d.batch, d.H, d.P, d.N)))

    def token(self, rng):
        x, Bm, Cm, raw = super().token(rng)
        if self.kind == "rows":   # one row in eight is `big`, the others are smaller by any factor
            size = self.big * np.exp(-rng.uniform(0, 20.7, x.shape))
            size[..., ::8] = self.big
        else:                     # every other token is `big` and adds nothing: the state is the other tokens'
            size = self.big if self.made % 2 else 1e-3
            if self.made % 2:
                Bm = np.zeros_like(Bm)
        self.made += 1
        x = (np.sign(x.astype(np.float64)) * size * rng.uniform(0.5, 1, x.shape)).astype(np.float16)
        return x, Bm, (Cm.astype(np.float32) * 1e-2).astype(np.float16), raw


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("shape", [(2, 4, 64, 128, 1, 5), (1, 3, 64, 64, 1, 4), (1, 2, 48, 256, 1, 3), (1, 2, 64, 128, 1, 20),
                                   (2, 3, 75, 203, 1, 16), (1, 2, 20, 260, 2, 3)])
@pytest.mark.parametrize("kind,big", [("rows", 1000.0), ("rows", 30000.0), ("tokens", 30000.0)])
def test_rows_and_tokens_of_different_sizes(ctx, shape, bits, kind, big):
    """A row's digits do not depend on its neighbours', nor a token's on the others': the bounds of every other test."""
    rng = np.random.default_rng(shape[3] + bits)
    run_tokens(SizedTokens(ctx, dims(*shape, bits), rng, kind, big), rng, min(2 * shape[5] + 1, 40))


@pytest.mark.gpu
def test_two_threads_with_different_shapes(ctx):
    """A context a host thread, over shapes whose launches want different amounts of shared memory: no call of one is
    refused for the other's."""
    import threading

    failed, start = [], threading.Barrier(2)

    def work(P):
        try:
            c = lssm.Ctx(0)
            d = dims(1, 1, P, 255, 1, 20, 16)
            cache, ops = lssm.StateCache(c, d), lssm.Ops(c)
            A = lssm.DeviceBuffer.from_array(c, np.zeros(1, np.float16))
            out = lssm.DeviceBuffer(c, P * 255 * 2)
            start.wait()
            for _ in range(20):
                c.begin_batch()
                try:
                    for _ in range(300):
                        ops.state_cache_load(cache, A, out, lssm.DT_F16, d)
                finally:
                    c.commit_and_wait()
            c.close()
        except Exception as e:   # noqa: BLE001
            failed.append((P, repr(e)))
            start.abort()

    threads = [threading.Thread(target=work, args=(P,)) for P in (150, 255)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed

"""GPU: the engine's scoring calls (lssm_score, lssm_session_logprobs) and its decode over a quantised
state cache (session option "state_bits"), alone and together: scoring is how the cache's cost is seen.

Tolerances:
  * lssm_session_logprobs works on the very logits lssm_session_logits returns: the operator's own bound,
    (V / 256 + 64) 2^-24 plus the roundings of the values;
  * against the oracle, logits are within 0.1 (as in the other engine tests), so log probabilities are
    within 0.2: a log-sum-exp moves by at most as much as its largest argument;
  * two runs whose arithmetic differs in fp32 summation order only: logits within 2e-2 + 2e-3 |logit| (as
    persistent against per-op decode), log probabilities within twice that of the largest logit; between fp32
    and cached states logit_tol, which is worked out there. Decode over the cache is such a run until the first fold when the states start at zero (nothing is rounded), and with
    16 bits throughout: a rounding to 2^-16 of a row's maximum is 32 times finer than the fp16 roundings of
    the activations that the two runs share.
"""

import numpy as np
import pytest

import lssm
import pyoracle as po

pytestmark = pytest.mark.gpu


def hp_of(**kw):
    hp = dict(d_model=256, n_layer=3, d_state=128, d_conv=4, expand=2, vocab_size=1000, n_heads=8, d_head=64, chunk_size=64,
              n_groups=1, norm_before_gate=0)
    hp.update(kw)
    return hp


def make(ctx, seed=5, int4=True, **kw):
    hp = hp_of(**kw)
    return hp, lssm.Model.synthesize(ctx, lssm.hparams(**hp), seed=seed, int4=int4)


def log_softmax(x):
    x = np.asarray(x, np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def check_against_logits(logits, targets, got, k, slack=0.0):
    V = logits.shape[-1]
    lp = log_softmax(logits)
    E = (V / 256 + 64) * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(lp).max() + slack
    logp, ent = got[0], got[1]
    for b in range(len(targets)):
        want = 0.0 if targets[b] == lssm.NO_TOKEN else lp[b, targets[b]]
        assert abs(logp[b] - want) <= E
        assert abs(ent[b] + (np.exp(lp[b]) * lp[b]).sum()) <= E * (2 + abs(ent[b]) + np.log(V))
        if k and not slack:
            ids = np.lexsort((np.arange(V), -logits[b]))[:k]
            assert np.array_equal(got[2][b], ids)
            assert np.abs(got[3][b] - lp[b, ids]).max() <= E


@pytest.mark.parametrize("batch,persistent", [(1, 1), (2, 0), (5, 1)])
def test_session_logprobs_of_the_last_logits(ctx, batch, persistent):
    hp, m = make(ctx)
    rng = np.random.default_rng(batch)
    s = lssm.Session(ctx, m, batch=batch, max_seq_len=32)
    s.set_option("persistent", persistent)
    with pytest.raises(lssm.LssmError, match="no logits"):
        s.logprobs(np.zeros(batch), 3)
    cur = s.prefill(rng.integers(0, 1000, (batch, 19)))
    for step in range(3):
        t = rng.integers(0, 1000, batch).astype(np.uint32)
        t[0] = lssm.NO_TOKEN if step == 1 else t[0]
        check_against_logits(s.logits(), t, s.logprobs(t, 7), 7)
        assert len(s.logprobs(t)) == 2
        assert np.array_equal(s.logprobs(t, 1)[2][:, 0], cur)   # the greedy pick is the first alternative
        cur = s.decode(cur, 1)[:, 0]
    s.close()


@pytest.mark.parametrize("cfg,int4", [(dict(), True), (dict(d_state=32, vocab_size=333, n_groups=2), False)])
def test_score_matches_oracle(ctx, cfg, int4):
    hp, m = make(ctx, int4=int4, **cfg)
    V, L = hp["vocab_size"], 30
    tok = np.random.default_rng(1).integers(0, V, (1, L)).astype(np.uint32)
    s = lssm.Session(ctx, m, batch=1, max_seq_len=L)
    logp, ent, ids, top = s.score(tok, 4)
    ora = po.OracleModel(m.download_bytes(), mode=0)
    _, pre, steps = ora.generate(tok[0, :1], L, teacher=tok[0, 1:].tolist() + [0])
    rows = np.concatenate([pre[None], steps])[:L]   # the logits after each token
    lp = log_softmax(rows)
    assert np.abs(logp[0, :-1] - lp[np.arange(L - 1), tok[0, 1:]]).max() <= 0.2
    assert logp[0, -1] == 0.0
    # an entropy moves by at most sum |d(p log p)|: 0.2 (1 + max |log p + H|) weighted by p, below 0.2 (2 + log V)
    assert np.abs(ent[0] + (np.exp(lp) * lp).sum(1)).max() <= 0.2 * (2 + np.log(V))
    assert np.abs(top[0] - np.take_along_axis(lp, ids[0].astype(np.int64), 1)).max() <= 0.2
    assert (np.diff(top[0], axis=1) <= 0).all()
    s.close()


@pytest.mark.parametrize("batch,L", [(1, 1), (1, 40), (3, 7), (4, 33)])
def test_score_is_a_prefill_that_keeps_every_row(ctx, batch, L):
    """Against prefills of every prefix (the logits there come from the GEMV kernels), and the session goes on
    as after a prefill."""
    hp, m = make(ctx, seed=9)
    rng = np.random.default_rng(L)
    tok = rng.integers(0, 1000, (batch, L)).astype(np.uint32)
    s, q = (lssm.Session(ctx, m, batch=batch, max_seq_len=L) for _ in range(2))
    logp, ent = s.score(tok)
    assert logp.shape == (batch, L) and (logp[:, -1] == 0).all()
    for i in sorted({0, L // 2, L - 1}):
        q.reset()
        first = q.prefill(tok[:, :i + 1])
        lg = q.logits()
        lp = log_softmax(lg)
        tol = 2 * (2e-2 + 2e-3 * np.abs(lg).max())
        if i < L - 1:
            assert np.abs(logp[:, i] - lp[np.arange(batch), tok[:, i + 1]]).max() <= tol
        assert np.abs(ent[:, i] + (np.exp(lp) * lp).sum(1)).max() <= tol * (2 + np.log(1000))
    assert np.array_equal(s.logits(), lg)
    assert np.array_equal(s.decode(first, 4), q.decode(first, 4))
    s.close()
    q.close()


def test_score_in_runs_of_rows(ctx):
    """More rows than one run of logits holds (64 MiB of a 50288-token vocabulary: 640 rows)."""
    hp, m = make(ctx, n_layer=1, vocab_size=50288, d_model=64, n_heads=2)
    tok = np.random.default_rng(2).integers(0, 50288, (3, 300)).astype(np.uint32)
    s = lssm.Session(ctx, m, batch=3, max_seq_len=300)
    logp, ent, ids, top = s.score(tok, 2)
    one = lssm.Session(ctx, m, batch=1, max_seq_len=300)
    for b in range(3):
        l1, e1, i1, t1 = one.score(tok[b], 2)
        one.reset()
        tol = 2 * (2e-2 + 2e-3 * 20)
        assert np.abs(l1[0] - logp[b]).max() <= tol and np.abs(e1[0] - ent[b]).max() <= tol * (2 + np.log(50288))
        assert np.abs(t1[0] - top[b]).max() <= tol
    s.close()
    one.close()


def test_scoring_refusals(ctx):
    hp, m = make(ctx, n_layer=1)
    s = lssm.Session(ctx, m, batch=2, max_seq_len=8)
    L, tok = lssm.lib(), np.zeros(32, np.uint32)
    p, f = tok.ctypes.data_as(lssm.P), np.zeros(4096, np.float32)
    o = f.ctypes.data_as(lssm.P)

    def refused(match, st):
        assert st != 0
        with pytest.raises(lssm.LssmError, match=match):
            lssm.check(st)

    refused("null argument", L.lssm_score(None, p, 4, 0, o, None, None, None))
    refused("null argument", L.lssm_score(s.h, None, 4, 0, o, None, None, None))
    refused("L must be", L.lssm_score(s.h, p, 0, 0, o, None, None, None))
    refused("exceeds", L.lssm_score(s.h, p, 9, 0, o, None, None, None))
    refused("top_k must be", L.lssm_score(s.h, p, 4, 33, o, o, p, o))
    refused("top_ids", L.lssm_score(s.h, p, 4, 2, o, o, None, o))
    refused("top_ids", L.lssm_score(s.h, p, 4, 0, o, o, p, None))
    refused("no output", L.lssm_score(s.h, p, 4, 0, None, None, None, None))
    refused("null session", L.lssm_session_logprobs(None, p, 0, o, None, None, None))
    refused("no logits", L.lssm_session_logprobs(s.h, p, 0, o, None, None, None))
    refused("needs targets", L.lssm_session_logprobs(s.h, None, 0, o, None, None, None))
    with pytest.raises(lssm.LssmError, match="out of range"):
        s.score(np.full((2, 4), 1000))
    s.score(np.zeros((2, 4)))   # the session is usable
    lssm.check(L.lssm_session_logprobs(s.h, None, 0, None, o, None, None))   # entropy needs no targets
    ctx.begin_batch()
    try:
        refused("batch is active", L.lssm_score(s.h, p, 4, 0, o, None, None, None))
        refused("batch is active", L.lssm_session_logprobs(s.h, p, 0, o, None, None, None))
        for key, value in (("state_bits", 8), ("state_window", 4)):
            with pytest.raises(lssm.LssmError, match="batch is active"):
                s.set_option(key, value)
    finally:
        ctx.commit_and_wait()
    for key, bad in (("state_bits", 4), ("state_bits", 32), ("state_window", 0), ("state_window", 33)):
        with pytest.raises(lssm.LssmError, match=key):
            s.set_option(key, bad)
    s.close()


# ---- decode over the quantised cache ------------------------------------------------------------------

def logit_tol(lg, d_model=256):
    """Two runs that share every fp16 rounding but not the last bits of what is rounded (other summation order; dt by
    log1p here, by log(1 + e^x) in the fp32 step, which differ by less than 2^-14 of dt): single roundings fall the
    other way, and the inputs n_k of lm_head, rounded to fp16, are off by an ulp, 2^-10 of their size. Then
    |d logit| <= 2^-10 sum_k |n_k w_k| <= 2^-10 |n| |w| (Cauchy-Schwarz). With |n| = sqrt(d_model) (what an RMS norm
    gives) a logit n . w has the root mean square |w| over directions of n, so |w| is the logits' root mean square.
    The logit's own rounding adds an ulp of it."""
    return 2.0 ** -10 * (np.sqrt(d_model) * np.sqrt(np.mean(np.square(lg))) + np.abs(lg))


def close_logits(a, b):
    np.testing.assert_array_less(np.abs(a - b), logit_tol(b))


def forced(s, seq, n, start):
    """Teacher-forced decode of n tokens of `seq` from `start`: logits after each."""
    out = []
    for i in range(n):
        s.decode(seq[:, start + i], 1)
        out.append(s.logits())
    return np.stack(out)


CONFIGS = [dict(), dict(n_groups=2), dict(d_state=48, d_head=32, n_heads=16), dict(d_state=75)]


@pytest.mark.parametrize("cfg", CONFIGS)
@pytest.mark.parametrize("bits,window", [(8, 16), (16, 9)])
def test_cached_decode_from_zero_is_exact_until_a_fold(ctx, cfg, bits, window):
    hp, m = make(ctx, seed=3, **cfg)
    seq = np.random.default_rng(7).integers(0, 1000, (3, window)).astype(np.uint32)
    a, b = (lssm.Session(ctx, m, batch=3, max_seq_len=8) for _ in range(2))
    b.set_option("state_bits", bits)
    b.set_option("state_window", window)
    close_logits(forced(b, seq, window - 1, 0), forced(a, seq, window - 1, 0))
    a.close()
    b.close()


@pytest.mark.parametrize("cfg", CONFIGS)
@pytest.mark.parametrize("graph", [0, 1])
def test_cached_decode_16_bits(ctx, cfg, graph):
    """A prefill, 40 decode steps (several folds), a second prefill that takes the states back to fp32, more steps."""
    hp, m = make(ctx, seed=4, **cfg)
    rng = np.random.default_rng(8)
    a, b = (lssm.Session(ctx, m, batch=4, max_seq_len=24) for _ in range(2))
    for s in (a, b):
        s.set_option("cuda_graph", graph)
    b.set_option("state_bits", 16)
    prompt, seq, more = (rng.integers(0, 1000, (4, n)).astype(np.uint32) for n in (24, 45, 11))
    for s in (a, b):
        s.prefill(prompt)
    close_logits(forced(b, seq, 40, 0)[::13], forced(a, seq, 40, 0)[::13])
    for s in (a, b):
        s.prefill(more)
    close_logits(b.logits(), a.logits())
    close_logits(forced(b, seq, 5, 40), forced(a, seq, 5, 40))
    # and off again: the states go on in fp32
    b.set_option("state_bits", 0)
    close_logits(forced(b, seq, 3, 0), forced(a, seq, 3, 0))
    a.close()
    b.close()


def test_cached_decode_many_steps_in_one_call(ctx):
    """One lssm_decode of many steps (a replayed graph) equals the same steps one by one."""
    hp, m = make(ctx, seed=6)
    prompt = np.random.default_rng(9).integers(0, 1000, (3, 12)).astype(np.uint32)
    outs = []
    for chunks in ([37], [1] * 37, [20, 17]):
        s = lssm.Session(ctx, m, batch=3, max_seq_len=12)
        s.set_option("state_bits", 8)
        cur, got = s.prefill(prompt), []
        for n in chunks:
            t = s.decode(cur, n)
            got.append(t)
            cur = t[:, -1]
        outs.append((np.concatenate(got, 1), s.logits()))
        s.close()
    for t, lg in outs[1:]:
        assert np.array_equal(t, outs[0][0]) and np.array_equal(lg, outs[0][1])


def test_persistent_decode_keeps_fp32_states(ctx):
    """state_bits applies where the persistent kernel does not run; switching between the two moves the states."""
    hp, m = make(ctx, seed=2)
    prompt = np.random.default_rng(5).integers(0, 1000, (1, 16)).astype(np.uint32)
    seq = np.random.default_rng(6).integers(0, 1000, (1, 40)).astype(np.uint32)
    a, b = (lssm.Session(ctx, m, batch=1, max_seq_len=16) for _ in range(2))
    a.set_option("persistent", 0)
    b.set_option("state_bits", 16)
    for s in (a, b):
        s.prefill(prompt)
    close_logits(forced(b, seq, 4, 0), forced(a, seq, 4, 0))
    assert b.launches()[1] == 1
    b.set_option("persistent", 0)
    close_logits(forced(b, seq, 20, 4), forced(a, seq, 20, 4))
    assert b.launches()[1] > 1
    b.set_option("persistent", 1)
    close_logits(forced(b, seq, 4, 24), forced(a, seq, 4, 24))
    b.reset()
    a.reset()
    for s in (a, b):
        s.prefill(prompt)
    close_logits(forced(b, seq, 2, 0), forced(a, seq, 2, 0))
    a.close()
    b.close()


@pytest.mark.parametrize("bits", [8, 16])
def test_score_and_cached_decode_together(ctx, bits):
    """What a quantised cache costs a continuation: its tokens' log probabilities, scored with fp32 states in one
    prefill, and met one by one in a decode over the cache. 16 bits: the two-run tolerance. 8 bits: a fold rounds a
    row's elements by at most 2^-8 of the row's maximum, so an output of the layer moves by at most 2^-8 of what it
    would be with every state element at its row's maximum: with rows whose maximum is about 3 times their root mean
    square, and errors of random sign, a relative 3 / sqrt(3) 2^-8 of the layer's output per fold still remembered.
    The decays here forget within two windows, so 2 folds x 3 layers, each below 0.7 %: 4 % of the largest logit."""
    hp, m = make(ctx, seed=13)
    rng = np.random.default_rng(14)
    prompt, cont = rng.integers(0, 1000, (3, 20)).astype(np.uint32), rng.integers(0, 1000, (3, 36)).astype(np.uint32)
    whole = np.concatenate([prompt, cont], 1)
    a = lssm.Session(ctx, m, batch=3, max_seq_len=whole.shape[1])
    logp, ent, ids, top = a.score(whole, 3)
    b = lssm.Session(ctx, m, batch=3, max_seq_len=20)
    b.set_option("state_bits", bits)
    b.prefill(prompt)
    got = [b.logprobs(cont[:, 0], 3)]
    biggest = two = 0.0
    for i in range(cont.shape[1] - 1):
        b.decode(cont[:, i], 1)
        got.append(b.logprobs(cont[:, i + 1], 3))
        lg = b.logits()
        biggest, two = max(biggest, float(np.abs(lg).max())), max(two, float(logit_tol(lg).max()))
    lp = np.stack([g[0] for g in got], 1)
    want = logp[:, 19:-1]
    tol = 2 * two + (2 * 0.04 * biggest if bits == 8 else 0.0)
    worst = np.abs(lp - want).max()
    print(f"[cache] {bits} bits: worst |d logp| {worst:.4f} (tolerance {tol:.4f}), mean logp {want.mean():.4f} -> {lp.mean():.4f}")
    assert worst <= tol
    a.close()
    b.close()


def test_a_failed_decode_does_not_fail_the_next_call(ctx):
    """The error of a step that cannot be captured (the default stream) is reported once."""
    c = lssm.Ctx(0)
    c.set_stream(0)
    hp, m = make(c, seed=16)
    tok = np.random.default_rng(2).integers(0, 1000, (3, 6)).astype(np.uint32)
    s = lssm.Session(c, m, batch=3, max_seq_len=6)
    first = s.prefill(tok)
    with pytest.raises(lssm.LssmError, match="captur"):
        s.decode(first, 2)
    s.set_option("cuda_graph", 0)
    q = lssm.Session(c, m, batch=3, max_seq_len=6)
    q.set_option("cuda_graph", 0)
    assert np.array_equal(s.decode(first, 2), q.decode(q.prefill(tok), 2))
    s.close()
    q.close()
    c.close()


def test_failed_decode_leaves_the_states_where_they_were(ctx):
    """A decode that ends before the states are quantised (a step cannot be captured on the default stream): later calls
    go on from the states of the prefill."""
    c = lssm.Ctx(0)
    c.set_stream(0)
    hp, m = make(c, seed=17)
    rng = np.random.default_rng(3)
    prompt, seq = rng.integers(0, 1000, (3, 20)).astype(np.uint32), rng.integers(0, 1000, (3, 8)).astype(np.uint32)

    def session(fail):
        s = lssm.Session(c, m, batch=3, max_seq_len=20)
        s.set_option("state_bits", 8)
        s.prefill(prompt)
        if fail:
            with pytest.raises(lssm.LssmError):
                s.decode(seq[:, 0], 1)
        s.set_option("cuda_graph", 0)
        return s

    goes_on = [lambda s: forced(s, seq, 8, 0),                                  # a decode over the cache
               lambda s: (s.prefill(seq), s.logits())[1],                       # a prefill, from fp32 states
               lambda s: (s.set_option("state_bits", 16), forced(s, seq, 8, 0))[1],
               lambda s: s.score(seq)[0]]
    for go in goes_on:
        a, b = session(False), session(True)
        assert np.array_equal(go(b), go(a))
        a.close()
        b.close()
    c.close()


@pytest.mark.parametrize("batch,L", [(1, 1), (1, 40), (3, 33), (12, 5)])
def test_score_ends_with_the_logits_it_leaves(ctx, batch, L):
    """The last entry of every sequence is of the very logits that the session holds afterwards, and that the greedy
    pick was made of."""
    hp, m = make(ctx, seed=11)
    tok = np.random.default_rng(batch).integers(0, 1000, (batch, L)).astype(np.uint32)
    s = lssm.Session(ctx, m, batch=batch, max_seq_len=L)
    logp, ent, ids, top = s.score(tok, 6)
    _, e, i, t = s.logprobs(np.full(batch, lssm.NO_TOKEN, np.uint32), 6)
    assert np.array_equal(ent[:, -1], e) and np.array_equal(ids[:, -1], i) and np.array_equal(top[:, -1], t)
    assert np.array_equal(ids[:, -1, 0], s.logits().argmax(1)) and (logp[:, -1] == 0).all()
    only = s.score(tok)[1]   # a continuation: other numbers, the same rule, without alternatives
    assert np.array_equal(only[:, -1], s.logprobs(np.zeros(batch))[1])
    s.close()


@pytest.mark.parametrize("bits", [8, 16])
def test_cached_decode_of_a_tensor_parallel_session(ctx, bits):
    """A communicator of one rank: the sharded path over the cache, against its own fp32 states until the first fold and,
    with 16 bits, behind it, and back to fp32 before a prefill and by the option; with 8 bits, in one call or in several."""
    hp, m = make(ctx, seed=19, n_groups=2)
    rng = np.random.default_rng(5)
    prompt, seq, more = (rng.integers(0, 1000, (3, n)).astype(np.uint32) for n in (16, 30, 9))
    comm = lssm.Comm(ctx, 0, 1, bytes(lssm.COMM_ID_BYTES))
    a, b = (lssm.Session(ctx, m, batch=3, max_seq_len=16, comm=comm) for _ in range(2))
    b.set_option("state_bits", bits)
    b.set_option("state_window", 7)
    close_logits(forced(b, seq, 6, 0), forced(a, seq, 6, 0))   # from zero: nothing is rounded before the fold
    for s in (a, b):
        s.reset()
        s.prefill(prompt)
    if bits == 16:
        close_logits(forced(b, seq, 25, 0), forced(a, seq, 25, 0))
        for s in (a, b):
            s.prefill(more)
        close_logits(forced(b, seq, 3, 25), forced(a, seq, 3, 25))
        b.set_option("state_bits", 0)
        close_logits(forced(b, seq, 3, 0), forced(a, seq, 3, 0))
    else:   # folds at different places of a call, captured or not
        one = lssm.Session(ctx, m, batch=3, max_seq_len=16, comm=comm)
        one.set_option("state_bits", 8)
        one.set_option("state_window", 7)
        one.set_option("cuda_graph", 0)
        cur = one.prefill(prompt)
        for s in (one, b):
            s.reset()
            s.prefill(prompt)
        first, second = b.decode(cur, 9), one.decode(cur, 20)
        assert np.array_equal(np.concatenate([first, b.decode(first[:, -1], 11)], 1), second)
        assert np.array_equal(b.logits(), one.logits())
        one.close()
    a.close()
    b.close()


def test_cached_decode_on_another_stream_than_the_option(ctx):
    """Setting state_bits leaves nothing under way on the context's stream that a decode on the next one could meet."""
    import torch

    c = lssm.Ctx(0)
    hp, m = make(c, seed=23)
    rng = np.random.default_rng(1)
    prompt, seq = rng.integers(0, 1000, (48, 6)).astype(np.uint32), rng.integers(0, 1000, (48, 4)).astype(np.uint32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for switch in (False, True, True):
        c.set_stream(streams[0].cuda_stream)
        s = lssm.Session(c, m, batch=48, max_seq_len=6)
        s.set_option("cuda_graph", 0)
        s.prefill(prompt)
        s.set_option("state_bits", 16)
        if switch:
            c.set_stream(streams[1].cuda_stream)
        outs.append(forced(s, seq, 4, 0))
        s.close()
    assert np.array_equal(outs[1], outs[0]) and np.array_equal(outs[2], outs[0])
    c.close()


def test_decode_after_a_history_that_did_not_fit(ctx):
    """A decode of more steps than device memory holds the tokens of is refused, and the next one runs."""
    hp, m = make(ctx, seed=29)
    tok = np.random.default_rng(6).integers(0, 1000, (16, 5)).astype(np.uint32)
    s, q = (lssm.Session(ctx, m, batch=16, max_seq_len=5) for _ in range(2))
    first = s.prefill(tok)
    s.decode(first, 2)
    st = lssm.lib().lssm_decode(s.h, first.ctypes.data_as(lssm.P), 0xFFFFFFFF, None)   # 16 * 2^32 * 4 bytes: 256 GiB
    assert st != 0
    cur = q.prefill(tok)
    q.decode(cur, 2)
    assert np.array_equal(s.decode(first, 2), q.decode(cur, 2))
    s.close()
    q.close()

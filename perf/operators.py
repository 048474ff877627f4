"""The measured cases of the scoring and state-cache operators, with their plain forms.

  logprobs       log probability of a given token, entropy, log-sum-exp and the top alternatives of rows of logits
  logprobs_grad  the gradient of log probability and entropy with respect to the logits
  state_step     one decode token of a batch of sequences over the quantised state cache, and the state read back
  state_park     a batch's states quantised into the cache and read back
"""

import math
import os
import sys

import torch

own = False

NONE = -1  # a row without a target token (0xFFFFFFFF as the library reads it)
FLOATS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"f16": 0, "bf16": 1, "f32": 2}


def listed():
    return [
        # one decode step's logits of a single sequence, with the 20 alternatives that a completion API returns
        dict(name="lp-decode-1row", kind="logprobs", rows=1, vocab=50288, dtype="f16", top_k=20, pad=0, masked=0.0),
        # a decode step of 64 sequences over the widest vocabulary, a few alternatives
        dict(name="lp-64rows-wide", kind="logprobs", rows=64, vocab=256000, dtype="f16", top_k=5, pad=0, masked=0.0),
        # scoring every token of a 2048-token prompt
        dict(name="lp-prompt-2048", kind="logprobs", rows=2048, vocab=50288, dtype="f16", top_k=20, pad=0, masked=0.0),
        # fp32 logits of constrained decoding: odd vocabulary, padded rows, most entries masked in some rows
        dict(name="lp-f32-masked", kind="logprobs", rows=333, vocab=32001, dtype="f32", top_k=8, pad=3, masked=0.9),
        # the loss gradient of a 2048-token prompt
        dict(name="grad-prompt-2048", kind="logprobs_grad", rows=2048, vocab=50288, dtype="f16", grad="f16", pad=0, masked=0.0, entropy=False),
        # the same with an entropy term on an odd vocabulary with padded rows and masked entries
        dict(name="grad-bf16-ragged", kind="logprobs_grad", rows=257, vocab=32001, dtype="bf16", grad="f32", pad=5, masked=0.5, entropy=True),
        # one layer of the 64-sequence batched decode
        dict(name="step-64seq-8bit", kind="state_step", batch=64, heads=80, headdim=64, dstate=128, groups=1, window=16, bits=8),
        # one layer of the 4-sequence decode with 8 groups, 16-bit codes
        dict(name="step-4seq-16bit", kind="state_step", batch=4, heads=128, headdim=64, dstate=128, groups=8, window=16, bits=16),
        # one layer of a small model, one sequence: latency
        dict(name="step-1seq-small", kind="state_step", batch=1, heads=24, headdim=64, dstate=128, groups=1, window=16, bits=8),
        # shapes outside the common ones: odd state size, short window
        dict(name="step-ragged", kind="state_step", batch=5, heads=12, headdim=48, dstate=75, groups=3, window=7, bits=16),
        # the states of 64 sequences parked in 8 bits and read back, one layer
        dict(name="park-64seq-8bit", kind="state_park", batch=64, heads=80, headdim=64, dstate=128, groups=1, window=16, bits=8, out="f32"),
        # one sequence's states parked in 16 bits and read back
        dict(name="park-1seq-16bit", kind="state_park", batch=1, heads=80, headdim=64, dstate=128, groups=1, window=16, bits=16, out="f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs_grad", "state_step", "state_park"])
    if kind in ("logprobs", "logprobs_grad"):
        vocab = _log_int(rng, 50, 256000)
        dtype = rng.choice(["f16", "bf16", "f32"])
        most = (100 << 20) if kind == "logprobs" else (90 << 20)
        if dtype == "f32":
            most //= 2
        rows = _log_int(rng, 1, max(1, min(4096, most // (vocab + 8))))
        c = dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, pad=rng.choice([0, 0, 1, 2, 8, 13]),
                 masked=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.99), 3)]))
        if kind == "logprobs":
            c["top_k"] = min(vocab, rng.choice([0, 1, rng.randint(2, 32), rng.randint(2, 32)]))
        else:
            c["grad"] = rng.choice([dtype, "f32"])
            c["entropy"] = rng.random() < 0.5
            if c["grad"] == "f32":
                c["rows"] = max(1, min(rows, (60 << 20) // (vocab + 8)))
        return c
    headdim, dstate = rng.choice([(64, 128), (64, 128), (rng.randint(4, 128), rng.randint(4, 256))])
    groups = rng.choice([1, 1, 2, 4, 8])
    heads = groups * _log_int(rng, 1, max(1, 128 // groups))
    batch = _log_int(rng, 1, max(1, min(96, (40 << 20) // (heads * headdim * dstate))))
    c = dict(kind=kind, batch=batch, heads=heads, headdim=headdim, dstate=dstate, groups=groups,
             window=rng.choice([16, 16, 32, rng.randint(1, 32)]), bits=rng.choice([8, 16]))
    if kind == "state_park":
        c["out"] = rng.choice(["f32", "f16", "bf16"])
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _logits(case, g):
    rows, vocab, dtype = case["rows"], case["vocab"], FLOATS[case["dtype"]]
    full = torch.empty(rows, vocab + case["pad"], dtype=dtype, device="cuda")
    x = full[:, :vocab]
    x.copy_(torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.5))
    peak = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
    x.scatter_add_(1, peak, torch.full((rows, 1), 9.0, device="cuda", dtype=dtype))
    if case["pad"]:
        full[:, vocab:] = float("nan")  # what lies behind a row is nobody's business
    if case["masked"] > 0:
        away = torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"]
        away.scatter_(1, peak, False)
        row = torch.arange(rows, device="cuda")[:, None]
        x.masked_fill_(away & (row % 4 == 1), float("-inf"))
        x.masked_fill_(away & (row % 4 == 3), torch.finfo(dtype).min)
        x.masked_fill_(row % 16 == 5, float("-inf"))  # a mask that leaves nothing
        x.masked_fill_((row % 16 == 9) & (torch.arange(vocab, device="cuda")[None] != vocab // 3), float("-inf"))
    anything = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    coin = torch.rand(rows, generator=g, device="cuda")
    t = torch.where(coin < 0.6, peak[:, 0], anything)
    if case["masked"] > 0:  # a target at the type's lowest value would outweigh every other row of a comparison
        t = torch.where(torch.arange(rows, device="cuda") % 4 == 3, peak[:, 0], t)
    if rows > 1:
        t = torch.where(coin > 0.95, torch.full_like(t, NONE), t)
    return full, x, t.to(torch.int32)


def _prepare_logprobs(case, g):
    rows, k = case["rows"], case["top_k"]
    full, x, t = _logits(case, g)
    f = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")  # noqa: E731
    return dict(case=case, full=full, x=x, t=t, logp=f(rows), entropy=f(rows), lse=f(rows), top_logp=f(rows, k),
                top_ids=torch.empty(rows, k, dtype=torch.int32, device="cuda"))


def _prepare_logprobs_grad(case, g):
    rows, vocab = case["rows"], case["vocab"]
    full, x, t = _logits(case, g)
    # what the forward call left: log-sum-exp and entropy of the rows, by 64-bit sums over slices of rows
    lse = torch.empty(rows, dtype=torch.float32, device="cuda")
    ent = torch.empty(rows, dtype=torch.float32, device="cuda")
    for r in range(0, rows, 256):
        z = x[r:r + 256].double()
        l = torch.logsumexp(z, 1)
        lp = z - l[:, None]
        e = lp.exp()
        lse[r:r + 256] = l.float()
        ent[r:r + 256] = -torch.where(e > 0, e * lp, 0.0).sum(1).float()
    ent = torch.where(torch.isinf(lse), 0.0, ent)
    gl = torch.rand(rows, generator=g, device="cuda").add_(0.5).mul_(-64.0)  # a scaled loss: -64 / token
    gh = torch.randn(rows, generator=g, device="cuda").mul_(8.0) if case["entropy"] else None
    out = torch.empty(rows, vocab, dtype=FLOATS[case["grad"]], device="cuda")
    return dict(case=case, full=full, x=x, t=t, lse=lse, entropy=ent, gl=gl, gh=gh, dx=out)


def _quantise(S, bits):
    """Codes and row scales of fp32 states (.., N). The quotients in 64 bits: half a step between two codes is a border."""
    q = 127.0 if bits == 8 else 32767.0
    scale = (S.abs().amax(-1).double() / q).float()
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, torch.zeros_like(scale), scale)
    by = scale.double()[..., None]
    code = torch.round(torch.where(by > 0, S / by, torch.zeros_like(by))).clamp_(-q, q)
    return code.to(torch.int8 if bits == 8 else torch.int16), scale


def _states(case, g):
    B, H, P, N = case["batch"], case["heads"], case["headdim"], case["dstate"]
    S = torch.randn(B, H, P, N, generator=g, device="cuda")
    return S.mul_(torch.randn(B, H, P, 1, generator=g, device="cuda").exp_())


def _prepare_state_step(case, g):
    B, H, P, N, G, W = (case[k] for k in ("batch", "heads", "headdim", "dstate", "groups", "window"))
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    A_log = torch.log(1.0 + 15.0 * torch.rand(H, generator=g, device="cuda")).half()
    bias = (r(H) * 0.7 - 4.0).half()
    codes, scales = _quantise(_states(case, g), case["bits"])
    # sequences that joined the batch at different times: their windows are filled differently
    fill = ((torch.arange(B, device="cuda") * 5 + W - 1) % W).to(torch.int32)[:, None].expand(B, H).contiguous()
    dt = torch.nn.functional.softplus(r(B, H, W) * 0.5 - 4.0)
    return dict(case=case, codes=codes, scales=scales, fill=fill, win_dt=dt, win_x=r(B, W, H, P).half(), win_B=r(B, W, G, N).half(),
                x=r(B, H, P).half(), B=r(B, G, N).half(), C=r(B, G, N).half(), dt_raw=(r(B, H) * 0.5).half(), bias=bias, A_log=A_log,
                D=torch.rand(H, generator=g, device="cuda").half(), y=torch.empty(B, H, P, dtype=torch.float16, device="cuda"),
                state=torch.empty(B, H, P, N, dtype=torch.float16, device="cuda"))


def _prepare_state_park(case, g):
    B, H, P, N, G, W = (case[k] for k in ("batch", "heads", "headdim", "dstate", "groups", "window"))
    e = lambda dt, *s: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
    return dict(case=case, S=_states(case, g), A_log=torch.zeros(H, dtype=torch.float16, device="cuda"),
                codes=e(torch.int8 if case["bits"] == 8 else torch.int16, B, H, P, N), scales=e(torch.float32, B, H, P),
                fill=torch.zeros(B, H, dtype=torch.int32, device="cuda"), win_dt=e(torch.float32, B, H, W), win_x=e(torch.float16, B, W, H, P),
                win_B=e(torch.float16, B, W, G, N), out=e(FLOATS[case["out"]], B, H, P, N))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"logprobs": _prepare_logprobs, "logprobs_grad": _prepare_logprobs_grad, "state_step": _prepare_state_step,
            "state_park": _prepare_state_park}[case["kind"]](case, g)


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _plain_logprobs(s):
    z, t, k = s["x"].float(), s["t"].long(), s["case"]["top_k"]
    rows, vocab = z.shape
    m = z.amax(1, keepdim=True)
    base = torch.where(torch.isinf(m), torch.zeros_like(m), m)  # a row with nothing left
    d = z - base
    e = torch.exp(d)
    total = e.sum(1)
    u = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1)
    log_total = torch.log(total)
    lse = base[:, 0] + log_total
    entropy = torch.where(total > 0, log_total - u / total, torch.zeros_like(total))
    xt = z.gather(1, t.clamp(min=0)[:, None])[:, 0]
    logp = torch.where(t == NONE, torch.zeros_like(lse), torch.where(torch.isinf(lse), lse, (xt - base[:, 0]) - log_total))
    if k == 0:
        return dict(logp=logp, entropy=entropy, lse=lse)
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)  # whole numbers in the order of the values
    key = order * vocab + (vocab - 1 - torch.arange(vocab, device=z.device))  # of equal values the lower index first
    ids = vocab - 1 - torch.topk(key, k, 1).values % vocab
    tops = z.gather(1, ids)
    top_logp = torch.where(torch.isinf(lse)[:, None], lse[:, None].expand_as(tops), (tops - base) - log_total[:, None])
    return dict(logp=logp, entropy=entropy, lse=lse, top_ids=ids.to(torch.int32), top_logp=top_logp)


def _plain_logprobs_grad(s):
    z, t = s["x"].float(), s["t"].long()
    empty = torch.isinf(s["lse"])[:, None]
    lp = z - torch.where(empty, torch.zeros_like(s["lse"][:, None]), s["lse"][:, None])
    p = torch.exp(lp)
    has = (t != NONE)[:, None]
    hot = (torch.arange(z.shape[1], device=z.device)[None] == t[:, None]) & has
    gl = torch.where(has, s["gl"][:, None], torch.zeros_like(s["gl"][:, None]))
    d = gl * (hot.float() - p)
    if s["gh"] is not None:
        d = d - s["gh"][:, None] * torch.where(p > 0, p * (lp + s["entropy"][:, None]), torch.zeros_like(p))
    return dict(dx=torch.where(empty, torch.zeros_like(d), d).to(s["dx"].dtype))


def _plain_state_step(s):
    c = s["case"]
    B, H, P, N, G, W = (c[k] for k in ("batch", "heads", "headdim", "dstate", "groups", "window"))
    a = -torch.exp(s["A_log"].float())
    raw = s["dt_raw"].float() + s["bias"].float()
    dt = torch.clamp(torch.where(raw > 20, raw, torch.log1p(torch.exp(raw))), 1e-6, 1e6)
    n = s["fill"][:, 0].long()
    rows = torch.arange(B, device=n.device)
    s["win_x"][rows, n] = s["x"]
    s["win_B"][rows, n] = s["B"]
    s["win_dt"][rows, :, n] = dt
    there = (torch.arange(W, device=n.device)[None] <= n[:, None])[:, None]  # (B, 1, W)
    wdt = torch.where(there, s["win_dt"], torch.zeros_like(s["win_dt"]))
    steps = a[None, :, None] * wdt
    upto = steps.flip(-1).cumsum(-1).flip(-1)
    alpha = torch.exp(upto[..., 0])
    w = wdt * torch.exp(upto - steps)  # (B, H, W)
    X = torch.where(there[..., None], s["win_x"].float().transpose(1, 2), torch.zeros((), device=n.device)) * w[..., None]  # (B, H, W, P)
    Bw = torch.where(there[..., None], s["win_B"].float().transpose(1, 2), torch.zeros((), device=n.device))  # (B, G, W, N)
    S = (s["codes"].float() * (s["scales"] * alpha[..., None])[..., None]).view(B, G, H // G, P, N)
    S = S + (X.transpose(2, 3).reshape(B, G, (H // G) * P, W) @ Bw).view(B, G, H // G, P, N)
    y = (S @ s["C"].float().view(B, G, 1, N, 1)).view(B, H, P) + s["D"].float()[None, :, None] * s["x"].float()
    S = S.view(B, H, P, N)
    full = n + 1 == W
    codes, scales = _quantise(S, c["bits"])
    s["codes"].copy_(torch.where(full[:, None, None, None], codes, s["codes"]))
    s["scales"].copy_(torch.where(full[:, None, None], scales, s["scales"]))
    s["fill"].copy_(torch.where(full, torch.zeros_like(n), n + 1)[:, None].expand(B, H))
    held = torch.where(full[:, None, None, None], codes.float() * scales[..., None], S)
    return dict(y=y.half(), state=held.half())


def _plain_state_park(s):
    codes, scales = _quantise(s["S"], s["case"]["bits"])
    s["codes"].copy_(codes)
    s["scales"].copy_(scales)
    s["fill"].zero_()
    return dict(scales=scales, state=(codes.float() * scales[..., None]).to(s["out"].dtype))


# ---- the framework's calls ------------------------------------------------------------------------------------------

_made = {}


def _ops():
    """The program's context of the current device and stream: on torch's stream, in a batch, so that calls are only enqueued."""
    device = torch._C._cuda_getDevice()
    at = (device, torch._C._cuda_getCurrentRawStream(device))  # as torch.cuda.current_stream().cuda_stream, in 0.3 us for 4
    if at not in _made:
        here = os.path.join(os.getcwd(), "lite-ssm_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import lssm

        ctx = lssm.Ctx(at[0])
        ctx.set_stream(at[1])
        ctx.begin_batch()
        _made[at] = lssm, ctx, lssm.Ops(ctx)
    return _made[at]


def _view(lssm, ctx, t):
    return None if t is None else lssm.DeviceView(ctx, t.data_ptr())


def _own_logprobs(s):
    lssm, ctx, ops = _ops()
    c, v = s["case"], lambda n: _view(lssm, ctx, s[n])  # noqa: E731
    k = c["top_k"]
    ops.logprobs(v("full"), v("t"), v("logp"), v("entropy"), v("lse"), v("top_ids") if k else None, v("top_logp") if k else None,
                 lssm.LogprobsDims(c["rows"], c["vocab"], k, CODES[c["dtype"]], c["vocab"] + c["pad"]))
    got = dict(logp=s["logp"], entropy=s["entropy"], lse=s["lse"])
    return dict(got, top_ids=s["top_ids"], top_logp=s["top_logp"]) if k else got


def _own_logprobs_grad(s):
    lssm, ctx, ops = _ops()
    c, v = s["case"], lambda n: _view(lssm, ctx, s[n])  # noqa: E731
    ops.logprobs_backward(v("full"), v("t"), v("lse"), v("entropy"), v("gl"), v("gh"), v("dx"),
                          lssm.LogprobsGradDims(c["rows"], c["vocab"], CODES[c["dtype"]], CODES[c["grad"]], c["vocab"] + c["pad"], c["vocab"]))
    return dict(dx=s["dx"])


def _cache(lssm, ctx, s):
    c = s["case"]
    dims = lssm.StateCacheDims(c["batch"], c["heads"], c["headdim"], c["dstate"], c["groups"], c["window"], c["bits"], 1e-6, 1e6, 1)
    return dims, lssm.StateCache.wrap(*(s[n].data_ptr() for n in ("codes", "scales", "win_x", "win_B", "win_dt", "fill")))


def _own_state_step(s):
    lssm, ctx, ops = _ops()
    v = lambda n: _view(lssm, ctx, s[n])  # noqa: E731
    dims, cache = _cache(lssm, ctx, s)
    ops.ssd_step_cached(v("x"), v("B"), v("C"), v("dt_raw"), v("bias"), v("A_log"), v("D"), cache, v("y"), dims)
    ops.state_cache_load(cache, v("A_log"), v("state"), lssm.DT_F16, dims)
    return dict(y=s["y"], state=s["state"])


def _own_state_park(s):
    lssm, ctx, ops = _ops()
    v = lambda n: _view(lssm, ctx, s[n])  # noqa: E731
    dims, cache = _cache(lssm, ctx, s)
    ops.state_cache_store(v("S"), cache, dims)
    ops.state_cache_load(cache, v("A_log"), v("out"), CODES[s["case"]["out"]], dims)
    return dict(scales=s["scales"], state=s["out"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"logprobs": _own_logprobs, "logprobs_grad": _own_logprobs_grad, "state_step": _own_state_step, "state_park": _own_state_park}[kind](state)
    return {"logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad, "state_step": _plain_state_step, "state_park": _plain_state_park}[kind](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (16 + 8 * case["top_k"]), "flops": 6 * n}
    if case["kind"] == "logprobs_grad":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (SIZE[case["dtype"]] + SIZE[case["grad"]]) + 20 * case["rows"], "flops": 5 * n}
    B, H, P, N, G, W = (case[k] for k in ("batch", "heads", "headdim", "dstate", "groups", "window"))
    n, code = B * H * P * N, case["bits"] // 8
    if case["kind"] == "state_park":
        return {"bytes": n * (4 + code + SIZE[case["out"]]) + 4 * B * H * P, "flops": 4 * n}
    fills = [(b * 5 + W - 1) % W for b in range(B)]
    window = sum(f + 1 for f in fills) * (2 * H * P + 2 * G * N + 4 * H)
    folds = sum(f + 1 == W for f in fills) / B
    return {"bytes": n * (code + 2) + folds * n * code + 4 * B * H * P + window + B * (4 * H * P + 4 * G * N),
            "flops": n * 2 + 2 * H * P * N * sum(f + 1 for f in fills)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("logprobs", "logprobs_grad"):
        parts = []
        for r in range(0, case["rows"], 128):
            x, t = s["x"][r:r + 128].double(), s["t"][r:r + 128].long()
            lse = torch.logsumexp(x, 1)
            none_left = torch.isneginf(lse)
            lp = torch.where(none_left[:, None], float("-inf"), x - torch.where(none_left, 0.0, lse)[:, None])
            p = torch.exp(lp)
            share = torch.where(torch.isneginf(lp), 0.0, p * torch.where(torch.isneginf(lp), 0.0, lp))
            H = -share.sum(1)
            given = t >= 0
            at = t.clamp(min=0)
            if case["kind"] == "logprobs":
                one = dict(logp=torch.where(given, lp[torch.arange(len(t)), at], 0.0), entropy=H, lse=lse)
                if case["top_k"]:
                    # the values alone: which index comes first among equals does not change them
                    one["top_logp"] = torch.sort(lp, 1, descending=True).values[:, :case["top_k"]].clone()
                parts.append(one)
            else:
                g = torch.where(given, s["gl"][r:r + 128].double(), 0.0)
                d = -g[:, None] * p
                d[torch.arange(len(t)), at] += torch.where(none_left, 0.0, g)
                if s["gh"] is not None:
                    d -= s["gh"][r:r + 128].double()[:, None] * (share + p * H[:, None])
                parts.append(dict(dx=torch.where(none_left[:, None], 0.0, d)))
        got = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
        return dict(got, top_ids=None) if case["kind"] == "logprobs" and case["top_k"] else got
    top = 127 if case["bits"] == 8 else 32767

    def held(S):  # what a state stands for once it is held in codes
        scale = (S.abs().max(-1, keepdim=True).values / top).float().double()  # the scale is held in 32 bits
        return torch.where(scale > 0, torch.round(S / torch.where(scale > 0, scale, 1.0)) * scale, 0.0), scale[..., 0]

    if case["kind"] == "state_park":
        got = [held(s["S"][b].double()) for b in range(case["batch"])]
        return dict(scales=torch.stack([g[1] for g in got]), state=torch.stack([g[0].to(torch.float64) for g in got]))
    # one sequence after the other, token by token, as the recurrence is written
    ys, states = [], []
    per = case["heads"] // case["groups"]
    A = -torch.exp(s["A_log"].double())
    for b in range(case["batch"]):
        S = s["codes"][b].double() * s["scales"][b].double()[..., None]
        n = int(s["fill"][b, 0])
        for j in range(n + 1):
            if j < n:
                x, k, dt = s["win_x"][b, j].double(), s["win_B"][b, j].double(), s["win_dt"][b, :, j].double()
            else:
                x, k = s["x"][b].double(), s["B"][b].double()
                dt = torch.nn.functional.softplus(s["dt_raw"][b].double() + s["bias"].double()).clamp(1e-6, 1e6)
            k = k.repeat_interleave(per, 0)
            S = torch.exp(A * dt)[:, None, None] * S + (dt[:, None] * x)[..., None] * k[:, None, :]
        C = s["C"][b].double().repeat_interleave(per, 0)
        ys.append((S * C[:, None, :]).sum(-1) + s["D"].double()[:, None] * s["x"][b].double())
        states.append(held(S)[0] if n + 1 == case["window"] else S)
    return dict(y=torch.stack(ys), state=torch.stack(states))

"""A gated recurrent block and the head of a token policy, as measurable cases.

Log probabilities of given tokens with the entropy and the top alternatives
(``token_log_probs``: a rollout step, and a learner's minibatch forward and
backward), a gated linear recurrence (``gated_scan``: training sequences and
prompts; ``gated_scan_step``: one rollout step) and the norms around a block
with its gate and residual scale (``residual_norm``).

Where ``own`` is false, ``run`` computes them from elementary torch operations
in float32; ``exact`` restates them in float64 from their definitions.
"""
from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------- the cases
def _case(name, defaults, kw):
    case = dict(defaults)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _tokens(name, kind, **kw):
    return _case(name, {"kind": kind, "rows": 1, "vocab": 2, "dtype": "bfloat16", "mask": "none", "padding": 0.0,
                        "temperature": 1.0, "top": 0, "sliced": False}, kw)


def _gated(name, kind, **kw):
    return _case(name, {"kind": kind, "batch": 1, "steps": 1, "features": 1, "dtype": "bfloat16", "done": 0.0,
                        "ragged": False, "carry": True, "packed": False}, kw)


def _residual(name, kind, **kw):
    return _case(name, {"kind": kind, "batch": 1, "steps": 1, "width": 1, "dtype": "bfloat16", "stream": "bfloat16",
                        "gate": "none", "post_norm": True, "packed": False}, kw)


def listed():
    return [
        # the action of each env of a small rollout step, illegal actions masked: bound by the call
        _tokens("tokens_step_few", "tokens", rows=16, vocab=43, dtype="float32", mask="rows"),
        # a serving step of a token policy: few rows of a large vocabulary, with alternatives
        _tokens("tokens_step_vocab", "tokens", rows=32, vocab=131072, top=8, temperature=0.8),
        # a learner's minibatch over a discrete action space, illegal actions masked, both passes
        _tokens("tokens_train_actions", "tokens_train", rows=262144, vocab=43, dtype="float32", mask="rows"),
        # sequences of tokens padded to one length, a vocabulary no vector divides, the last step's logits left out
        _tokens("tokens_train_vocab", "tokens_train", rows=8192, vocab=50001, padding=0.2, sliced=True),
        # a rollout step of a few envs: bound by the call
        _gated("gated_step", "gated_step", batch=64, features=1000, done=0.02),
        # one long context
        _gated("gated_prompt_long", "gated", batch=1, steps=65536, features=2048, packed=True),
        # a recurrent learner's sequence minibatch: 256 envs x 64 steps, 256 features, episode resets, both passes
        _gated("gated_train_f32", "gated_train", batch=256, steps=64, features=256, dtype="float32", done=0.02),
        # long training sequences of unequal lengths with resets, features in parts of one projection's output
        _gated("gated_train_ragged", "gated_train", batch=24, steps=4093, features=640, done=0.005, ragged=True,
               packed=True),
        # a rollout step's rows between two blocks
        _residual("residual_step", "residual", batch=64, width=1000),
        # the rows of the long context, a float32 stream
        _residual("residual_prompt", "residual", batch=1, steps=65536, width=2048, stream="float32"),
        # of training sequences, gates through a sigmoid, both passes
        _residual("residual_train_gate", "residual_train", batch=128, steps=1000, width=640, gate="sigmoid", packed=True),
        # a width no vector divides, plain gates, no norm of the block's output, both passes
        _residual("residual_train_odd", "residual_train", batch=48, steps=333, width=1333, dtype="float32",
                  stream="float32", gate="plain", post_norm=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tokens", "tokens", "tokens_train", "tokens_train", "gated", "gated_train", "gated_train",
                       "gated_step", "residual", "residual_train", "residual_train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    while True:
        if kind in ("tokens", "tokens_train"):
            rows, vocab = _log_int(rng, 1, 262144), _log_int(rng, 2, 262144)
            if rows * vocab <= 1 << 28:
                return _tokens(None, kind, rows=rows, vocab=vocab, dtype=dtype, mask=rng.choice(["none", "none", "rows", "one"]),
                               padding=rng.choice([0.0, 0.2]), temperature=rng.choice([1.0, 1.0, 0.7, 1.3]),
                               top=min(vocab, rng.choice([0, 0, 1, 5, 8, 20])) if rows * vocab <= 1 << 25 else 0,
                               sliced=rng.random() < 0.3)
        elif kind == "gated_step":
            batch, features = _log_int(rng, 1, 4096), _log_int(rng, 16, 8192)
            return _gated(None, kind, batch=batch, features=features, dtype=dtype, done=rng.choice([0.0, 0.03]))
        elif kind in ("gated", "gated_train"):
            batch, steps, features = _log_int(rng, 1, 512), _log_int(rng, 1, 65536), _log_int(rng, 16, 8192)
            if batch * steps * features <= (1 << 27 if kind == "gated" else 1 << 26):
                return _gated(None, kind, batch=batch, steps=steps, features=features, dtype=dtype,
                              done=rng.choice([0.0, 0.002, 0.03]), ragged=steps > 1 and rng.random() < 0.3,
                              carry=rng.random() < 0.7, packed=rng.random() < 0.5)
        else:
            batch, steps, width = _log_int(rng, 1, 512), _log_int(rng, 1, 65536), _log_int(rng, 16, 8192)
            if batch * steps * width <= (1 << 27 if kind == "residual" else 1 << 26):
                return _residual(None, kind, batch=batch, steps=steps, width=width, dtype=dtype,
                                 stream=rng.choice([dtype, "float32"]), gate=rng.choice(["none", "plain", "sigmoid"]),
                                 post_norm=rng.random() < 0.7, packed=rng.random() < 0.5)


# ---------------------------------------------------------------------- inputs
def _dtype(name):
    return F32 if name == "float32" else torch.bfloat16


def _normal(gen, *shape, dtype=F32):
    return torch.randn(*shape, device=DEV, dtype=F32, generator=gen).to(dtype)


def _parts(case, gen, count, lead, width, dtype):
    """`count` tensors [*lead, width]: of their own, or (packed) parts of one projection's output."""
    if not case["packed"]:
        return [_normal(gen, *lead, width, dtype=dtype) for _ in range(count)]
    whole = _normal(gen, *lead, -(-count * width // 64) * 64, dtype=dtype)
    return [whole[..., i * width:(i + 1) * width] for i in range(count)]


def _prepare_tokens(case, gen, s):
    rows, vocab = case["rows"], case["vocab"]
    # two rows a sequence where that divides: (sliced) the logits of one step more are left out
    steps = 2 if rows % 2 == 0 else 1
    lead = (rows // steps, steps + (1 if case["sliced"] else 0))
    logits = (2.5 * _normal(gen, *lead, vocab)).to(_dtype(case["dtype"]))
    s["logits"] = logits[:, :-1] if case["sliced"] else logits
    lead = (rows // steps, steps)
    s["tokens"] = torch.randint(0, vocab, lead, device=DEV, generator=gen)
    s["mask"] = None
    if case["mask"] == "rows":
        s["mask"] = torch.rand(*lead, vocab, device=DEV, generator=gen) < 0.7
        s["mask"].scatter_(-1, s["tokens"][..., None], True)
        # an env that has ended has no legal action
        s["mask"][torch.rand(lead, device=DEV, generator=gen) < 0.02] = False
    elif case["mask"] == "one":
        s["mask"] = torch.rand(vocab, device=DEV, generator=gen) < 0.9
    if case["padding"]:
        s["tokens"] = torch.where(torch.rand(lead, device=DEV, generator=gen) < case["padding"], -1, s["tokens"])
    if case["dtype"] == "float32":
        s["tokens"] = s["tokens"].int()
    if case["kind"] == "tokens_train":
        s["dlog_prob"], s["dentropy"] = _normal(gen, *lead), 0.01 * _normal(gen, *lead)
        s["logits"] = s["logits"].detach().requires_grad_()
    return s


def _prepare_gated(case, gen, s):
    B, T, F, dt = case["batch"], case["steps"], case["features"], _dtype(case["dtype"])
    step = case["kind"] == "gated_step"
    s["x"], s["input_gate"], s["decay_gate"] = _parts(case, gen, 3, (B,) if step else (B, T), F, dt)
    # rates from 0.02 to 2 over the features: time constants of one step to a hundred
    s["rate"] = torch.exp(torch.empty(F, device=DEV).uniform_(math.log(0.02), math.log(2.0), generator=gen))
    s["carry0"] = _normal(gen, B, F) if case["carry"] else None
    done = torch.rand(B, T, device=DEV, generator=gen) < case["done"]
    s["done"] = None if case["done"] == 0 else done[:, 0] if step else done
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(T // 2, T + 1, (B,), device=DEV, dtype=torch.int32, generator=gen)
        s["lengths"][0] = T
    if case["kind"] == "gated_train":
        s["dout"], s["dfinal"] = _normal(gen, B, T, F, dtype=dt), _normal(gen, B, F)
        for n in ("x", "input_gate", "decay_gate", "rate", "carry0"):
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
    return s


def _prepare_residual(case, gen, s):
    B, T, D = case["batch"], case["steps"], case["width"]
    dt, stream = _dtype(case["dtype"]), _dtype(case["stream"])
    s["block"], s["gate"] = _parts(case, gen, 2, (B, T), D, dt)
    s["gate_name"] = case["gate"]
    if case["gate"] == "none":
        s["gate"] = None
    s["residual"] = (3 * _normal(gen, B, T, D)).to(stream)
    s["post_scale"] = 1 + 0.1 * _normal(gen, D) if case["post_norm"] else None
    s["pre_scale"], s["residual_scale"] = 1 + 0.1 * _normal(gen, D), 0.5 + 0.1 * _normal(gen, D)
    if case["kind"] == "residual_train":
        s["dstream"], s["dnormed"] = _normal(gen, B, T, D, dtype=stream), _normal(gen, B, T, D, dtype=dt)
        for n in ("block", "gate", "residual", "post_scale", "pre_scale", "residual_scale"):
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["kind"].startswith("tokens"):
        return _prepare_tokens(case, gen, s)
    if case["kind"].startswith("gated"):
        return _prepare_gated(case, gen, s)
    return _prepare_residual(case, gen, s)


# ----------------------------------------------------------------- plain forms
def _plain_tokens(s):
    dt, T = s["logits"].dtype, s["temperature"]
    x = s["logits"].detach().float()
    if s["mask"] is not None:
        x = torch.where(s["mask"], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    w = (x - torch.where(m == -math.inf, 0.0, m)) / T
    e = torch.exp(w)
    total = e.sum(-1, keepdim=True)
    none = total == 0
    log_total = torch.log(torch.where(none, 1.0, total))
    # log p; every entry of a row without any is -inf
    w = w - log_total
    p = e / torch.where(none, 1.0, total)
    entropy = -torch.where(p > 0, p * w, 0.0).sum(-1)
    inside = (s["tokens"] >= 0) & (s["tokens"] < s["vocab"])
    at = torch.where(inside, s["tokens"], 0).long()[..., None]
    log_prob = torch.where(inside, w.gather(-1, at)[..., 0], 0.0)
    got = {"log_prob": log_prob, "entropy": entropy}
    if s["kind"] == "tokens_train":
        g = torch.where(inside & (log_prob > -math.inf), s["dlog_prob"], 0.0)[..., None]
        h = s["dentropy"][..., None]
        d = -p * (g + h * torch.where(p > 0, w + entropy[..., None], 0.0))
        got["dlogits"] = (d.scatter_add_(-1, at, g) / T).to(dt)
    if s["top"]:
        place = torch.arange(s["vocab"], device=x.device)
        values, indices = [], []
        for _ in range(s["top"]):
            best = x.amax(-1, keepdim=True)
            i = torch.where(x == best, place, s["vocab"]).amin(-1, keepdim=True)
            values.append(w.gather(-1, i))
            indices.append(torch.where(best == -math.inf, -1, i))
            x = x.scatter(-1, i, -math.inf)
        got["top_log_probs"] = torch.where(torch.cat(indices, -1) < 0, -math.inf, torch.cat(values, -1))
        got["top_tokens"] = torch.cat(indices, -1).to(s["tokens"].dtype)
    return got


def _plain_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from h_{-1} = 0: maps of spans that double."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _plain_gates(x, input_gate, decay_gate, rate):
    i, r = torch.sigmoid(input_gate), torch.sigmoid(decay_gate)
    log_a = -rate * r
    return i, r, log_a, torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a))


def _plain_gated(s):
    dt = s["x"].dtype
    x, ig, dg = (s[n].detach().float() for n in ("x", "input_gate", "decay_gate"))
    rate, carry = s["rate"].detach(), s["carry0"]
    i, r, log_a, a, w = _plain_gates(x, ig, dg, rate)
    if s["kind"] == "gated_step":
        kept = carry if s["done"] is None else torch.where(s["done"][:, None], 0.0, carry)
        h = a * kept + w * i * x
        return {"carry": h, "out": h.to(dt)}
    B, T, F = x.shape
    inside = torch.ones(B, T, 1, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        inside = (torch.arange(T, device=x.device) < s["lengths"][:, None])[..., None]
    kept = inside if s["done"] is None else inside & ~s["done"][..., None]
    decay = torch.where(inside, torch.where(kept, a, 0.0), 1.0)
    first = torch.zeros(B, F, device=x.device) if carry is None else carry.detach()
    b = torch.where(inside, w * i * x, 0.0)
    b[:, 0] += decay[:, 0] * first
    h = _plain_scan(decay, b)
    got = {"carry": h[:, -1].clone(), "out": torch.where(inside, h, 0.0).to(dt)}
    if s["kind"] == "gated_train":
        g = torch.where(inside, s["dout"].float(), 0.0)
        g[:, -1] += s["dfinal"]
        after = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], 1)
        d = _plain_scan(after.flip(1), g.flip(1)).flip(1)
        if carry is not None:
            got["dcarry"] = d[:, 0] * decay[:, 0]
        d = torch.where(inside, d, 0.0)
        before = torch.where(kept, torch.cat([first[:, None], h[:, :-1]], 1), 0.0)
        dlog_a = d * (a * before - a * a * i * x / w)
        got["dx"], got["dinput_gate"] = (d * w * i).to(dt), (d * w * x * i * (1 - i)).to(dt)
        got["ddecay_gate"], got["drate"] = (dlog_a * log_a * (1 - r)).to(dt), -(dlog_a * r).sum((0, 1))
    return got


def _plain_residual(s):
    train, dt, stream = s["kind"] == "residual_train", s["block"].dtype, s["residual"].dtype
    names = [n for n in ("block", "gate", "residual", "post_scale", "pre_scale", "residual_scale") if s[n] is not None]
    leaves = {n: s[n].detach().float().requires_grad_(train) for n in names}
    with torch.set_grad_enabled(train):
        n = leaves["block"]
        if s["post_norm"]:
            n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + EPS) * leaves["post_scale"]
        if s["gate"] is not None:
            n = n * (torch.sigmoid(leaves["gate"]) if s["gate_name"] == "sigmoid" else leaves["gate"])
        y = leaves["residual"] + leaves["residual_scale"] * n
        z = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * leaves["pre_scale"]
    got = {"stream": y.detach().to(stream), "normed": z.detach().to(dt)}
    if train:
        grads = torch.autograd.grad([y, z], list(leaves.values()), [s["dstream"].float(), s["dnormed"].float()])
        got.update({"d" + n: x.to(s[n].dtype) for n, x in zip(names, grads)})
    return got


def _run_plain(s):
    if s["kind"].startswith("tokens"):
        return _plain_tokens(s)
    if s["kind"].startswith("gated"):
        return _plain_gated(s)
    return _plain_residual(s)


# ------------------------------------------------------------------------- run
def _run_own(s):
    from boonta_amd.kernels import gated_scan, gated_scan_step, residual_norm, token_log_probs
    kind = s["kind"]
    if kind.startswith("tokens"):
        o = token_log_probs(s["logits"], s["tokens"], s["mask"], temperature=s["temperature"], top=s["top"])
        got = {"log_prob": o.log_prob.detach(), "entropy": o.entropy.detach()}
        if s["top"]:
            got.update(top_log_probs=o.top_log_probs, top_tokens=o.top_tokens)
        if kind == "tokens_train":
            got["dlogits"], = torch.autograd.grad([o.log_prob, o.entropy], [s["logits"]], [s["dlog_prob"], s["dentropy"]])
        return got
    if kind == "gated_step":
        carry, out = gated_scan_step(s["x"], s["input_gate"], s["decay_gate"], s["rate"], s["carry0"], done=s["done"])
        return {"carry": carry, "out": out}
    if kind.startswith("gated"):
        carry, out = gated_scan(s["x"], s["input_gate"], s["decay_gate"], s["rate"], carry=s["carry0"], done=s["done"],
                                lengths=s["lengths"])
        got, outs, cots = {"carry": carry.detach(), "out": out.detach()}, [carry, out], ["dfinal", "dout"]
        names = ("x", "input_gate", "decay_gate", "rate", "carry0")
    else:
        outs = residual_norm(s["block"], s["residual"], gate=s["gate"], post_scale=s["post_scale"],
                             residual_scale=s["residual_scale"], pre_scale=s["pre_scale"], post_norm=s["post_norm"],
                             gate_activation="sigmoid" if s["gate_name"] == "sigmoid" else None, epsilon=EPS)
        got, cots = {"stream": outs[0].detach(), "normed": outs[1].detach()}, ["dstream", "dnormed"]
        names = ("block", "gate", "residual", "post_scale", "pre_scale", "residual_scale")
    if kind.endswith("train"):
        names = [n for n in names if s[n] is not None]
        grads = torch.autograd.grad(outs, [s[n] for n in names], [s[n] for n in cots])
        got.update({"dcarry" if n == "carry0" else "d" + n: x for n, x in zip(names, grads)})
    return got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    train = case["kind"].endswith("train")
    if case["kind"].startswith("tokens"):
        n = case["rows"] * case["vocab"]
        mask = n if case["mask"] == "rows" else 0
        # both passes need the logits; the second writes their gradient
        return {"bytes": n * e * (3 if train else 1) + mask * (2 if train else 1) + case["rows"] * (12 + 12 * case["top"]),
                "flops": n * (14 if train else 6)}
    if case["kind"].startswith("gated"):
        n = case["batch"] * case["steps"] * case["features"]
        read = 0.75 if case["ragged"] else 1.0      # rows past a sequence's length are not read
        state = 4 * case["batch"] * case["features"]
        flags = case["batch"] * case["steps"] if case["done"] > 0 else 0
        total = n * e * (3 * read + 1) + flags + state * (2 if case["carry"] else 1)
        if train:
            total += n * e * (4 * read + 3) + flags + state * (3 if case["carry"] else 1)
        return {"bytes": total, "flops": n * read * (50 if train else 15)}
    n = case["batch"] * case["steps"] * case["width"]
    r = 4 if case["stream"] == "float32" else 2
    gate = 0 if case["gate"] == "none" else 1
    total = n * (e * (2 + gate) + 2 * r)
    if train:
        # the block's output, gate and stream in, the two cotangents in, the gradients out
        total += n * (e * (3 + 2 * gate) + 3 * r)
    return {"bytes": total, "flops": n * (35 if train else 10)}


# ----------------------------------------------------------------------- exact
def _exact_tokens(s):
    V, T, k = s["vocab"], s["temperature"], s["top"]
    logits, tokens = s["logits"].detach().reshape(-1, V), s["tokens"].reshape(-1).long()
    n, train = tokens.numel(), s["kind"] == "tokens_train"
    shape = tuple(s["tokens"].shape)
    log_prob, entropy = (torch.zeros(n, dtype=F64, device=DEV) for _ in range(2))
    grad = torch.zeros(n, V, dtype=F64, device=DEV) if train else None
    best, which = torch.zeros(n, k, dtype=F64, device=DEV), torch.zeros(n, k, dtype=torch.long, device=DEV)
    many = max(1, (1 << 26) // V)
    for r0 in range(0, n, many):
        r = slice(r0, min(n, r0 + many))
        x = logits[r].double() / T
        if s["mask"] is not None:
            x = x.masked_fill(~s["mask"].expand(*shape, V).reshape(-1, V)[r], -math.inf)
        lse = torch.logsumexp(x, -1, keepdim=True)
        some = lse > -math.inf
        logp = torch.where(some, x - lse, -math.inf)
        p = logp.exp()
        H = -torch.special.xlogy(p, p).sum(-1)
        given = (tokens[r] >= 0) & (tokens[r] < V)
        hot = (torch.arange(V, device=DEV) == tokens[r][:, None]) & given[:, None]
        lp = torch.where(hot, logp, 0.0).sum(-1)
        log_prob[r], entropy[r] = lp, H
        if train:
            g = torch.where(given & (lp > -math.inf), s["dlog_prob"].reshape(-1)[r].double(), 0.0)[:, None]
            h = s["dentropy"].reshape(-1)[r].double()[:, None]
            d = torch.where(hot, g, 0.0) - g * p - h * (torch.special.xlogy(p, p) + p * H[:, None])
            grad[r] = d / T
        if k:
            # the sort keeps the order of equal values
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
            best[r] = logp.gather(-1, order)
            which[r] = torch.where(best[r] == -math.inf, -1, order)
    got = {"log_prob": log_prob.view(shape), "entropy": entropy.view(shape)}
    if train:
        got["dlogits"] = grad.view(*shape, V)
    if k:
        got.update(top_log_probs=best.view(*shape, k), top_tokens=which.view(*shape, k))
    return got


def _exact_gated(s):
    """Step after step."""
    step, train = s["kind"] == "gated_step", s["kind"] == "gated_train"
    x, ig, dg = (s[n].detach().double() for n in ("x", "input_gate", "decay_gate"))
    done = s["done"]
    if step:
        x, ig, dg, done = x[:, None], ig[:, None], dg[:, None], None if done is None else done[:, None]
    B, T, F = x.shape
    rate = s["rate"].detach().double()
    i, r = 1 / (1 + torch.exp(-ig)), 1 / (1 + torch.exp(-dg))
    a = torch.exp(-rate * r)
    w = torch.sqrt(-torch.expm1(-2 * rate * r))
    keep = torch.ones(B, T, dtype=F64, device=DEV) if done is None else (~done).double()
    lengths = torch.full((B,), T, device=DEV) if s["lengths"] is None else s["lengths"].long()
    inside = torch.arange(T, device=DEV) < lengths[:, None]
    a_kept = torch.where(inside[..., None], a * keep[..., None], 1.0)
    u = torch.where(inside[..., None], w * i * x, 0.0)
    h = torch.zeros(B, F, dtype=F64, device=DEV) if s["carry0"] is None else s["carry0"].detach().double()
    first, hs = h, torch.empty_like(u)
    for t in range(T):
        h = torch.addcmul(u[:, t], a_kept[:, t], h, out=hs[:, t])
    got = {"carry": hs[:, -1].clone(), "out": hs * inside[..., None]}
    if step:
        got["out"] = got["out"][:, 0]
    if train:
        g = s["dout"].double() * inside[..., None]
        d, D = s["dfinal"].double(), torch.empty_like(g)
        for t in range(T - 1, -1, -1):
            D[:, t] = g[:, t] + d
            d = a_kept[:, t] * D[:, t]
        if s["carry0"] is not None:
            got["dcarry"] = d
        D = D * inside[..., None]
        hs = torch.cat([first[:, None], hs[:, :-1]], 1) * keep[..., None]
        got["dx"], got["dinput_gate"] = D * w * i, D * w * x * i * (1 - i)
        # d h_t / d r = -rate a h_{t-1} + rate a^2 i x / w
        dr = D * rate * (a * a * i * x / w - a * hs)
        got["ddecay_gate"], got["drate"] = dr * r * (1 - r), (dr * r).sum((0, 1)) / rate
    return got


def _exact_residual(s):
    D = s["width"]
    u, x = s["block"].detach().double(), s["residual"].detach().double()
    wz, c = s["pre_scale"].detach().double(), s["residual_scale"].detach().double()
    g, dg = torch.ones((), dtype=F64, device=DEV), None
    if s["gate"] is not None:
        g = s["gate"].detach().double()
        if s["gate_name"] == "sigmoid":
            g = 1 / (1 + torch.exp(-g))
            dg = g * (1 - g)
    un, n = u, u
    if s["post_norm"]:
        ru = (u.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
        un = u * ru
        n = un * s["post_scale"].detach().double()
    y = x + c * g * n
    ry = (y.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
    got = {"stream": y, "normed": y * ry * wz}
    if s["kind"] == "residual_train":
        dy, dz = s["dstream"].double(), s["dnormed"].double()
        got["dpre_scale"] = (dz * y * ry).sum((0, 1))
        e = dz * wz
        dy = dy + ry * e - y * ry.pow(3) * (e * y).mean(-1, keepdim=True)
        got["dresidual"], got["dresidual_scale"] = dy, (dy * g * n).sum((0, 1))
        if s["gate"] is not None:
            got["dgate"] = dy * c * n * (1 if dg is None else dg)
        dn = dy * c * g
        got["dblock"] = dn
        if s["post_norm"]:
            got["dpost_scale"] = (dn * un).sum((0, 1))
            dn = dn * s["post_scale"].detach().double()
            got["dblock"] = ru * dn - u * ru.pow(3) * (dn * u).mean(-1, keepdim=True)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("tokens"):
        return _exact_tokens(s)
    return _exact_gated(s) if case["kind"].startswith("gated") else _exact_residual(s)

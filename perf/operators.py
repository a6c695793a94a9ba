"""The matrix-state recurrence of a recurrent torso and what makes its queries and keys, as measurable cases.

Linear attention with a decay for each head (``linear_attention``: the chunked
form of training minibatches and prompts, forward and backward;
``linear_attention_step``: one rollout step) and the per-head norms of queries
and keys with the position rotation (``qk_norm_rotary``).

Where ``own`` is false, ``run`` computes them from elementary torch operations
in float32 (rotation angles in float64); ``exact`` restates them in float64
from their definitions.
"""
from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------- the cases
def _attend(name, kind, **kw):
    case = {"kind": kind, "batch": 1, "steps": 1, "heads": 1, "kv_heads": 0, "key_dim": 64, "value_dim": 64,
            "dtype": "bfloat16", "done": 0.0, "ragged": False, "carry": True, "packed": False}
    case.update(kw)
    case["kv_heads"] = case["kv_heads"] or case["heads"]
    if name:
        case["name"] = name
    return case


def _norm(name, kind, **kw):
    case = {"kind": kind, "batch": 1, "steps": 1, "heads": 1, "kv_heads": 0, "dim": 64, "rotary": 64,
            "interleaved": False, "dtype": "bfloat16", "first": 0, "packed": False}
    case.update(kw)
    case["kv_heads"] = case["kv_heads"] or case["heads"]
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a rollout step of a few envs: bound by the call
        _attend("step_few_envs", "step", batch=16, heads=4, key_dim=64, value_dim=64, dtype="float32", done=0.02),
        # a rollout step of many envs with wide heads: the float32 states are read and written once
        _attend("step_many_envs", "step", batch=1024, heads=8, key_dim=128, value_dim=128, done=0.02),
        # a short evaluation prompt in float32, heads no tile divides, key heads shared by two
        _attend("prompt_short_odd", "attend", batch=4, steps=37, heads=6, kv_heads=3, key_dim=20, value_dim=33,
                dtype="float32", done=0.03),
        # prompts of unequal lengths in one padded batch, two query heads to a key head
        _attend("prompt_ragged", "attend", batch=24, steps=1531, heads=8, kv_heads=4, ragged=True),
        # one long context on few heads
        _attend("prompt_long", "attend", batch=1, steps=65536, heads=16, key_dim=128, value_dim=128, packed=True),
        # a recurrent learner's sequence minibatch: 256 envs x 64 steps, four heads of 64 in place of a 256-wide GRU
        _attend("train_minibatch_f32", "train", batch=256, steps=64, heads=4, dtype="float32", done=0.02),
        # long training sequences with episode resets, 512 features in eight heads, steps no chunk divides
        _attend("train_resets_bf16", "train", batch=128, steps=1000, heads=8, done=0.005, packed=True),
        # the largest training batch
        _attend("train_wide_bf16", "train", batch=8, steps=4096, heads=16, key_dim=128, value_dim=128, carry=False),
        # the queries and keys of one rollout step, far into an episode
        _norm("norm_step", "norm", batch=16, heads=4, dim=64, rotary=64, dtype="float32", first=100000),
        # the queries and keys of the long context, taken from one projection's output
        _norm("norm_prompt", "norm", batch=1, steps=65536, heads=16, dim=128, rotary=128, packed=True),
        # of the training sequences, forward and backward
        _norm("norm_train_bf16", "norm_train", batch=128, steps=1000, heads=8, dim=64, rotary=64, packed=True),
        # neighbouring columns paired, part of an odd head rotated, shared key heads
        _norm("norm_train_odd", "norm_train", batch=48, steps=333, heads=6, kv_heads=2, dim=75, rotary=40,
              interleaved=True, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_DIMS = [16, 20, 32, 33, 48, 64, 64, 80, 96, 100, 128, 128]


def _draw_heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8])
    return kv * rng.choice([1, 1, 1, 2, 4]), kv


def draw(rng):
    kind = rng.choice(["step", "attend", "attend", "train", "train", "norm", "norm_train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    while True:
        heads, kv = _draw_heads(rng)
        if kind in ("norm", "norm_train"):
            dim = rng.choice(_DIMS + [192, 256])
            rotary = rng.choice([dim // 2 * 2, dim // 2 * 2, dim // 4 * 2, 0])
            steps, batch = _log_int(rng, 1, 16384), _log_int(rng, 1, 512)
            if batch * steps * (heads + kv) * dim <= (1 << 27 if kind == "norm" else 1 << 26):
                return _norm(None, kind, batch=batch, steps=steps, heads=heads, kv_heads=kv, dim=dim, rotary=rotary,
                             interleaved=rng.random() < 0.3, dtype=dtype, first=rng.choice([0, 0, 1 << 17]),
                             packed=rng.random() < 0.5)
            continue
        key_dim = rng.choice(_DIMS)
        value_dim = key_dim if rng.random() < 0.7 else rng.choice(_DIMS)
        wide = max(key_dim, value_dim)
        kw = {"heads": heads, "kv_heads": kv, "key_dim": key_dim, "value_dim": value_dim, "dtype": dtype,
              "done": rng.choice([0.0, 0.002, 0.03])}
        if kind == "step":
            batch = _log_int(rng, 1, 4096)
            if batch * heads * key_dim * value_dim <= 1 << 27:
                return _attend(None, "step", batch=batch, **kw)
            continue
        steps, batch = _log_int(rng, 1, 32768), _log_int(rng, 1, 512)
        fits = batch * steps * heads * wide <= (1 << 26 if kind == "attend" else 1 << 25)
        if fits and batch * heads * key_dim * value_dim <= 1 << 26:
            return _attend(None, kind, batch=batch, steps=steps, ragged=steps > 1 and rng.random() < 0.25,
                           carry=rng.random() < 0.7, packed=rng.random() < 0.5, **kw)


# ---------------------------------------------------------------------- inputs
def _dtype(case):
    return F32 if case["dtype"] == "float32" else torch.bfloat16


def _columns(case, gen, widths, lead):
    """Tensors [*lead, heads, width]: of their own, or (packed) parts of one projection's output."""
    dt = _dtype(case)
    if not case["packed"]:
        return [torch.randn(*lead, h, d, device=DEV, dtype=F32, generator=gen).to(dt) for h, d in widths]
    total = sum(h * d for h, d in widths)
    pitch = -(-total // 64) * 64
    whole = torch.randn(*lead, pitch, device=DEV, dtype=F32, generator=gen).to(dt)
    parts, at = [], 0
    for h, d in widths:
        parts.append(whole[..., at:at + h * d].unflatten(-1, (h, d)))
        at += h * d
    return parts


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, T, H, G = case["batch"], case["steps"], case["heads"], case["kv_heads"]
    dt = _dtype(case)
    s = dict(case)
    if case["kind"] in ("norm", "norm_train"):
        D = case["dim"]
        s["q"], s["k"] = _columns(case, gen, [(H, D), (G, D)], (B, T))
        s["q_scale"] = 1 + 0.1 * torch.randn(D, device=DEV, generator=gen)
        s["k_scale"] = 1 + 0.1 * torch.randn(D, device=DEV, generator=gen)
        s["positions"] = (case["first"] + torch.arange(T, device=DEV, dtype=torch.int32)
                          + torch.randint(0, 1000, (B, 1), device=DEV, dtype=torch.int32, generator=gen))
        pair = torch.arange(case["rotary"] // 2, device=DEV, dtype=F64)
        s["frequencies"] = 10000.0 ** (-2 * pair / max(1, case["rotary"]))
        if case["kind"] == "norm_train":
            s["dq"] = torch.randn(B, T, H, D, device=DEV, generator=gen).to(dt)
            s["dk"] = torch.randn(B, T, G, D, device=DEV, generator=gen).to(dt)
            for n in ("q", "k", "q_scale", "k_scale"):
                s[n] = s[n].detach().requires_grad_()
        return s
    K, V = case["key_dim"], case["value_dim"]
    # time constants from 32 to 512 steps over the heads
    s["log_decay"] = torch.log1p(-torch.exp(torch.linspace(math.log(1 / 32), math.log(1 / 512), H, device=DEV)))
    done = torch.rand(B, T, device=DEV, generator=gen) < case["done"]
    s["carry0"] = torch.randn(B, H, K, V, device=DEV, generator=gen) if case["carry"] else None
    if case["kind"] == "step":
        q, k, v = _columns(dict(case, packed=False), gen, [(H, K), (G, K), (G, V)], (B,))
        return dict(s, q=q, k=k, v=v, done=done[:, 0])
    s["done"] = done if case["done"] > 0 else None
    s["q"], s["k"], s["v"] = _columns(case, gen, [(H, K), (G, K), (G, V)], (B, T))
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(T // 2, T + 1, (B,), device=DEV, dtype=torch.int32, generator=gen)
        s["lengths"][0] = T
    if case["kind"] == "train":
        s["dout"] = torch.randn(B, T, H, V, device=DEV, generator=gen).to(dt)
        s["dfinal"] = torch.randn(B, H, K, V, device=DEV, generator=gen)
        for n in ("q", "k", "v", "carry0"):
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
    return s


# ----------------------------------------------------------------- plain forms
def _plain_attend(q, k, v, g, carry, done, lengths, scale):
    """float32 operands of full head counts, [batch, heads, steps, dim]; chunks of the steps side by side."""
    B, H, T, K = q.shape
    V = v.shape[-1]
    C = 64 if T <= 4096 else 256
    n = max(1, -(-T // C))
    pad = n * C - T
    t = torch.arange(n * C, device=q.device)
    ends = torch.full((B,), T, device=q.device) if lengths is None else lengths.long()
    valid = t < ends[:, None]
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)) for x in (q, k, v))
    k, v = (torch.where(valid[:, None, :, None], x, 0.0) for x in (k, v))
    episode = torch.zeros(B, n * C, dtype=torch.long, device=q.device)
    if done is not None:
        episode = (torch.nn.functional.pad(done, (0, pad)) & valid).long().cumsum(1)
    q, k, v = (x.unflatten(2, (n, C)) for x in (q, k, v))
    ep = episode.view(B, 1, n, C)
    last = ep[..., -1]                                                       # [B, 1, n]: the episode at a chunk's end
    before = torch.nn.functional.pad(last[..., :-1], (1, 0))                 # and at its start
    i = torch.arange(C, device=q.device)
    gap = (i[:, None] - i).clamp(min=0)
    decay = torch.where(i[:, None] >= i, torch.exp(g[:, None, None] * gap), 0.0)                   # [H, C, C]
    weights = torch.where(ep[..., :, None] == ep[..., None, :], decay[None, :, None], 0.0)
    out = (scale * (q @ k.transpose(-1, -2)) * weights) @ v
    count = (ends[:, None] - C * torch.arange(n, device=q.device)).clamp(0, C)[:, None]            # [B, 1, n]
    left = count[..., None] - 1 - i
    tail = torch.where((left >= 0) & (ep == last[..., None]), torch.exp(g[:, None, None] * left.clamp(min=0)), 0.0)
    states = ((k * tail[..., None]).transpose(-1, -2) @ v).flatten(-2)                             # [B, H, n, K V]
    at = torch.nn.functional.pad(count.cumsum(-1), (1, 0))                                         # [B, 1, n + 1]
    entered = torch.cat([before, last[..., -1:]], -1)                                              # episode entering c
    c = torch.arange(n + 1, device=q.device)
    between = (at[..., :, None] - at[..., None, 1:]).clamp(min=0)
    link = (c[:, None] > c[:-1]) & (entered[..., :, None] == last[..., None, :])
    states = torch.where(link, torch.exp(g[:, None, None] * between), 0.0) @ states                # [B, H, n + 1, K V]
    if carry is not None:
        first = torch.where(entered == 0, torch.exp(g[:, None] * at), 0.0)
        states = states + first[..., None] * carry.flatten(-2)[:, :, None]
    states = states.unflatten(-1, (K, V))
    reach = torch.where(ep == before[..., None], torch.exp(g[:, None, None] * (i + 1)), 0.0)
    out = out + scale * reach[..., None] * (q @ states[:, :, :-1])
    out = torch.where(valid[:, None, :, None], out.flatten(2, 3), 0.0)
    return states[:, :, -1], out[:, :, :T]


def _heads_first(x, group):
    return x.transpose(1, 2).repeat_interleave(group, dim=1)


def _run_plain(s):
    kind, group = s["kind"], s["heads"] // s["kv_heads"]
    if kind == "step":
        q, k, v = s["q"].float(), s["k"].float().repeat_interleave(group, 1), s["v"].float().repeat_interleave(group, 1)
        state = torch.where(s["done"][:, None, None, None], 0.0, s["carry0"])
        state = torch.exp(s["log_decay"])[:, None, None] * state + k[..., :, None] * v[..., None, :]
        out = (q[..., None, :] @ state)[..., 0, :] * s["key_dim"] ** -0.5
        return {"carry": state, "out": out.to(s["q"].dtype)}
    if kind in ("norm", "norm_train"):
        return _run_plain_norm(s)
    dt = s["q"].dtype
    leaves = [None if s[n] is None else s[n].detach().float().requires_grad_(kind == "train")
              for n in ("q", "k", "v", "carry0")]
    with torch.set_grad_enabled(kind == "train"):
        q, k, v = leaves[0].transpose(1, 2), _heads_first(leaves[1], group), _heads_first(leaves[2], group)
        final, out = _plain_attend(q, k, v, s["log_decay"], leaves[3], s["done"], s["lengths"], s["key_dim"] ** -0.5)
        out = out.transpose(1, 2)
    got = {"carry": final.detach(), "out": out.detach().to(dt).contiguous()}
    if kind == "train":
        names = [n for n, x in zip(("dq", "dk", "dv", "dcarry"), leaves) if x is not None]
        grads = torch.autograd.grad([out, final], [x for x in leaves if x is not None], [s["dout"].float(), s["dfinal"]])
        got.update({n: x if n == "dcarry" else x.to(dt) for n, x in zip(names, grads)})
    return got


def _plain_norm(x, scale, cos, sin, interleaved):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * scale
    R = 2 * cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., R:]], -1)


def _run_plain_norm(s):
    train, dt = s["kind"] == "norm_train", s["q"].dtype
    angle = s["positions"].double()[..., None] * s["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()
    leaves = [s[n].detach().float().requires_grad_(train) for n in ("q", "k", "q_scale", "k_scale")]
    with torch.set_grad_enabled(train):
        outs = [_plain_norm(x, w, cos, sin, s["interleaved"]) for x, w in ((leaves[0], leaves[2]), (leaves[1], leaves[3]))]
    got = {"q": outs[0].detach().to(dt), "k": outs[1].detach().to(dt)}
    if train:
        grads = torch.autograd.grad(outs, leaves, [s["dq"].float(), s["dk"].float()])
        got.update(dq=grads[0].to(dt), dk=grads[1].to(dt), dq_scale=grads[2], dk_scale=grads[3])
    return got


# ------------------------------------------------------------------------- run
def _run_own(s):
    from boonta_amd.kernels import linear_attention, linear_attention_step, qk_norm_rotary
    if s["kind"] == "step":
        carry, out = linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["carry0"], done=s["done"])
        return {"carry": carry, "out": out}
    if s["kind"] in ("norm", "norm_train"):
        q, k = qk_norm_rotary(s["q"], s["k"], s["q_scale"], s["k_scale"], s["frequencies"], s["positions"],
                              epsilon=EPS, interleaved=s["interleaved"])
        got = {"q": q.detach(), "k": k.detach()}
        if s["kind"] == "norm_train":
            grads = torch.autograd.grad([q, k], [s[n] for n in ("q", "k", "q_scale", "k_scale")], [s["dq"], s["dk"]])
            got.update(dq=grads[0], dk=grads[1], dq_scale=grads[2], dk_scale=grads[3])
        return got
    carry, out = linear_attention(s["q"], s["k"], s["v"], s["log_decay"], carry=s["carry0"], done=s["done"],
                                  lengths=s["lengths"])
    got = {"carry": carry.detach(), "out": out.detach()}
    if s["kind"] == "train":
        leaves = [(n, s[m]) for n, m in (("dq", "q"), ("dk", "k"), ("dv", "v"), ("dcarry", "carry0")) if s[m] is not None]
        grads = torch.autograd.grad([out, carry], [x for _, x in leaves], [s["dout"], s["dfinal"]])
        got.update({n: x for (n, _), x in zip(leaves, grads)})
    return got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    B, T, H, G = case["batch"], case["steps"], case["heads"], case["kv_heads"]
    if case["kind"] in ("norm", "norm_train"):
        n = B * T * (H + G) * case["dim"]
        train = case["kind"] == "norm_train"
        return {"bytes": n * e * (5 if train else 2) + 4 * B * T, "flops": n * (20 if train else 7)}
    K, V = case["key_dim"], case["value_dim"]
    state = 4 * B * H * K * V
    read = 0.75 if case["ragged"] else 1.0      # rows past a sequence's length are not read
    inputs, out = B * T * (H * K + G * (K + V)) * e * read, B * T * H * V * e
    flops = B * T * H * K * V * read
    flags = B * T if case["done"] > 0 else 0
    if case["kind"] == "step":
        return {"bytes": 2 * state + inputs + out + B, "flops": 4 * flops}
    forward = inputs + out + flags + state * (2 if case["carry"] else 1)
    if case["kind"] == "attend":
        return {"bytes": forward, "flops": 4 * flops}
    backward = 2 * inputs + out * read + flags + state * (3 if case["carry"] else 1)
    return {"bytes": forward + backward, "flops": 14 * flops}


# ----------------------------------------------------------------------- exact
def _exact_attend(s):
    """From the sums over pairs of steps, rows of a block against every step before them."""
    B, T, H, G = s["batch"], s["steps"], s["heads"], s["kv_heads"]
    K, V, group, train = s["key_dim"], s["value_dim"], H // G, s["kind"] == "train"
    dev, scale = s["q"].device, s["key_dim"] ** -0.5
    g = s["log_decay"].double()
    out = torch.zeros(B, H, T, V, dtype=F64, device=dev)
    final = torch.zeros(B, H, K, V, dtype=F64, device=dev)
    grads = [torch.zeros(B, H, T, d, dtype=F64, device=dev) for d in (K, K, V)] if train else None
    dcarry = torch.zeros(B, H, K, V, dtype=F64, device=dev)
    rows = min(T, 1024)
    many = max(1, int(2e8 // (rows * T * H)))
    step = torch.arange(T, device=dev)
    for b0 in range(0, B, many):
        at = slice(b0, min(B, b0 + many))
        q, k, v = (s[n].detach()[at].double().permute(0, 2, 1, 3) for n in ("q", "k", "v"))
        k, v = (x[:, torch.arange(H, device=dev) // group] for x in (k, v))
        length = torch.full((q.shape[0],), T, device=dev) if s["lengths"] is None else s["lengths"][at].long()
        inside = step < length[:, None]                                                  # [b, T]
        k, v, q = (torch.where(inside[:, None, :, None], x, 0.0) for x in (k, v, q))
        start = torch.full_like(inside, -1, dtype=torch.long)                            # the last reset up to a step
        if s["done"] is not None:
            start = torch.where(s["done"][at] & inside, step, -1).cummax(1).values
        ended = start[:, -1]
        old = torch.zeros(q.shape[0], H, K, V, dtype=F64, device=dev)
        if s["carry0"] is not None:
            old = s["carry0"].detach()[at].double()
        fresh = torch.where((start < 0) & inside, 1.0, 0.0)[:, None] * torch.exp(g[:, None] * (step + 1))   # [b, H, T]
        keep = (inside & (step >= ended[:, None]))[:, None]
        tail = torch.where(keep, torch.exp(g[:, None] * (length[:, None, None] - 1 - step).clamp(min=0)), 0.0)
        whole = torch.where((ended < 0)[:, None], torch.exp(g * length[:, None]), 0.0)[..., None, None]
        final[at] = (k * tail[..., None]).transpose(-1, -2) @ v + whole * old
        if train:
            do = torch.where(inside[:, None, :, None], s["dout"][at].double().permute(0, 2, 1, 3), 0.0)
            df = s["dfinal"][at].double()
            dq, dk, dv = (x[at] for x in grads)
            dk += tail[..., None] * (v @ df.transpose(-1, -2))
            dv += tail[..., None] * (k @ df)
            dq += scale * fresh[..., None] * (do @ old.transpose(-1, -2))
            dcarry[at] = whole * df + scale * (q * fresh[..., None]).transpose(-1, -2) @ do
        for r0 in range(0, T, rows):
            r, c = slice(r0, min(T, r0 + rows)), slice(0, min(T, r0 + rows))
            gap = step[r, None] - step[c]
            seen = (gap >= 0) & (step[c] >= start[:, r, None])                                     # [b, rows, steps]
            w = torch.where(seen[:, None], scale * torch.exp(g[:, None, None] * gap.clamp(min=0)), 0.0)
            p = (q[:, :, r] @ k[:, :, c].transpose(-1, -2)).mul_(w)
            out[at, :, r] = p @ v[:, :, c] + scale * fresh[:, :, r, None] * (q[:, :, r] @ old)
            if train:
                w.mul_(do[:, :, r] @ v[:, :, c].transpose(-1, -2))
                dq[:, :, r] += w @ k[:, :, c]
                dk[:, :, c] += w.transpose(-1, -2) @ q[:, :, r]
                dv[:, :, c] += p.transpose(-1, -2) @ do[:, :, r]
    got = {"carry": final, "out": out.transpose(1, 2)}
    if train:
        dq, dk, dv = grads
        got.update(dq=dq.transpose(1, 2), dk=dk.unflatten(1, (G, group)).sum(2).transpose(1, 2),
                   dv=dv.unflatten(1, (G, group)).sum(2).transpose(1, 2))
        if s["carry0"] is not None:
            got["dcarry"] = dcarry
    return got


def _exact_norm(s):
    train = s["kind"] == "norm_train"
    p = s["positions"].double()[:, :, None, None] * s["frequencies"]
    half = s["frequencies"].numel()
    pairs = torch.arange(half, device=DEV)
    first, second = (2 * pairs, 2 * pairs + 1) if s["interleaved"] else (pairs, pairs + half)
    got = {}
    for n in ("q", "k"):
        x, w = s[n].detach().double(), s[n + "_scale"].detach().double()
        r = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).pow(-0.5)
        y = w * (x * r)
        z = y.clone()
        z[..., first] = y[..., first] * torch.cos(p) - y[..., second] * torch.sin(p)
        z[..., second] = y[..., first] * torch.sin(p) + y[..., second] * torch.cos(p)
        got[n] = z
        if train:
            c = s["d" + n].double()
            e = c.clone()
            e[..., first] = c[..., first] * torch.cos(p) + c[..., second] * torch.sin(p)
            e[..., second] = c[..., second] * torch.cos(p) - c[..., first] * torch.sin(p)
            got["d" + n + "_scale"] = (e * x * r).sum((0, 1, 2))
            e = e * w
            got["d" + n] = r * e - x * r.pow(3) * (e * x).mean(-1, keepdim=True)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "norm_train"):
        return _exact_norm(s)
    if case["kind"] == "step":
        B, H, G, K, V = (case[n] for n in ("batch", "heads", "kv_heads", "key_dim", "value_dim"))
        of = torch.arange(H, device=DEV) // (H // G)
        state = s["carry0"].double() * s["log_decay"].double().exp()[:, None, None]
        state[s["done"]] = 0
        state.add_(s["k"].double()[:, of, :, None] * s["v"].double()[:, of, None, :])
        out = torch.stack([(s["q"].double()[..., None] * state)[..., j].sum(-1) for j in range(V)], -1)
        return {"carry": state, "out": out * K ** -0.5}
    return _exact_attend(s)

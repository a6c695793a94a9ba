"""The gated recurrence (sequences, gradients, one step) against the float64 oracle (oracle/gated.py).

Tolerances, N = 2^-24, gates' arguments up to 8: a sigmoid and what it leaves of 1 are
within 12 roundings,
so a = e^-q within 16 q + 4 of its value and b = w i x within 40 (w^2 = 1 - a^2 is at
worst 36 off, where the series gives way to the difference at 1/4).  The error of
a state follows the recurrence itself.  A state is a sum of terms, one of each
step before it, of sizes S_t = a_t S_{t-1} + |b_t|, and where maps are composed the
sum is cut between them: A h + B rounds to N |A h + B| <= N S_t, though A h and B
may cancel to a far smaller state, and A and B themselves are rounded sums and
products of those terms.  So each step adds at most N ((16 q + 4) a_t S_{t-1} + 40
|b_t|) in its chunk and as much again in the maps, e_t = a_t e_{t-1} + twice that,
and the maps of a tile (at most 3 of lanes, 8 of waves, 1 of its chunk) 12 N S_t.
The same holds for the cotangents of states, whose terms are |g_t|.  Gradients are
products of these: 60 roundings of the sizes of their terms and those errors.  A rate's gradient sums
steps x batch terms, (steps / 8 + batch + 64) roundings more of the sum of their
sizes.  bf16 outputs add their rounding, 2^-8 of the value."""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import gated_scan, gated_scan_step
from oracle import gated as og

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
N = 2.0 ** -24
NAMES = ("x", "input_gate", "decay_gate", "rate", "carry")


def np64(x):
    return x.detach().double().cpu().numpy()


def problem(seed, B, T, F, dtype, packed=False, done=0.0, ragged=False, carry=True):
    gen = torch.Generator().manual_seed(seed)
    if packed:
        whole = torch.randn(T, B, 3 * F + 5, generator=gen).to(dtype).cuda().transpose(0, 1)
        x, i, d = (whole[..., 1 + k * F:1 + (k + 1) * F] for k in range(3))
    else:
        x, i, d = (torch.randn(B, T, F, generator=gen).to(dtype).cuda() for _ in range(3))
    rate = torch.exp(torch.empty(F).uniform_(-5, 1, generator=gen)).cuda()
    ops = dict(x=x, input_gate=i, decay_gate=d, rate=rate, carry=torch.randn(B, F, generator=gen).cuda() if carry else None,
               done=(torch.rand(B, T, generator=gen) < done).cuda() if done else None, lengths=None)
    if ragged:
        ops["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32).cuda()
        ops["lengths"][0] = T
    return ops


def cotangents(seed, B, T, F, dtype):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(B, F, generator=gen).cuda(), torch.randn(B, T, F, generator=gen).to(dtype).cuda()


def run(ops, cots):
    leaves = {n: None if ops[n] is None else ops[n].detach().requires_grad_() for n in NAMES}
    outs = gated_scan(*leaves.values(), ops["done"], ops["lengths"])
    names = [n for n in NAMES if leaves[n] is not None]
    return outs, dict(zip(names, torch.autograd.grad(outs, [leaves[n] for n in names], list(cots))))


def within(got, want, tol):
    tol = tol + (2.0 ** -8 * np.abs(want) if got.dtype == BF16 else 1e-37)
    assert got.shape == want.shape and (np.abs(np64(got) - want) <= tol).all()


def check(ops, cots, outs, grads):
    x, i, d, rate = (np64(ops[n]) for n in NAMES[:4])
    B, T, F = x.shape
    carry = np.zeros((B, F)) if ops["carry"] is None else np64(ops["carry"])
    done = None if ops["done"] is None else ops["done"].cpu().numpy()
    lengths = None if ops["lengths"] is None else ops["lengths"].cpu().numpy()
    final, out, before = og.gated_scan(x, i, d, rate, carry, done, lengths)
    g = og.gates(x, i, d, rate)
    inside, kept = og._kept(x, done, lengths)
    a, q, b = g["a"], g["q"], np.abs(g["w"] * g["i"] * x)
    e, S, errors, entering = np.zeros((B, F)), np.abs(carry), np.zeros_like(x), np.zeros_like(x)
    for t in range(T):
        sizes = a[:, t] * np.where(kept[:, t], S, 0)
        entering[:, t] = np.where(kept[:, t], e + 12 * N * S, 0)
        new = a[:, t] * np.where(kept[:, t], e, 0) + 2 * N * ((16 * q[:, t] + 4) * sizes + 40 * b[:, t])
        e, S = np.where(inside[:, t], new, e), np.where(inside[:, t], sizes + b[:, t], S)
        errors[:, t] = np.where(inside[:, t], new + 12 * N * S, 0)
    within(outs[0], final, e + 12 * N * S)
    within(outs[1], out, errors)
    if grads is None:
        return
    dfinal, dout = np.zeros((B, F)) if cots[0] is None else np64(cots[0]), np.zeros_like(x) if cots[1] is None else np64(cots[1])
    want = og.gated_scan_vjp(x, i, d, rate, carry, done, lengths, dfinal, dout)
    D = want["D"]
    eE, S, eD = np.zeros((B, F)), np.abs(dfinal), np.zeros_like(x)
    for t in range(T - 1, -1, -1):
        sizes = S + np.abs(dout[:, t])
        eD[:, t] = np.where(inside[:, t], eE + 12 * N * sizes, 0)
        new = np.where(kept[:, t], a[:, t] * (eE + 2 * N * (16 * q[:, t] + 4) * sizes), 0)
        eE, S = np.where(inside[:, t], new, eE), np.where(inside[:, t], np.where(kept[:, t], a[:, t] * sizes, 0), S)
    size = np.abs(D) * 60 * N + eD
    u = np.abs(g["i"] * x)
    within(grads["x"], want["x"], size * g["w"] * g["i"])
    within(grads["input_gate"], want["input_gate"], size * g["w"] * u * (1 - g["i"]))
    slope = size * (np.abs(a * before) + a * a * u / g["w"]) + np.abs(D) * a * entering
    within(grads["decay_gate"], want["decay_gate"], slope * q * (1 - g["r"]))
    terms = np.abs(D) * (np.abs(a * before) + a * a * u / g["w"]) * g["r"]
    within(grads["rate"], want["rate"], (slope * g["r"] + (T / 8 + B + 64) * N * terms).sum((0, 1)))
    if "carry" in grads:
        within(grads["carry"], want["carry"], eE + 12 * N * S)


CASES = [  # batch, steps, features
    (1, 1, 1), (3, 1, 2), (2, 2, 3), (2, 3, 4), (2, 5, 7), (3, 8, 16), (1, 9, 5), (2, 31, 33), (2, 33, 64), (1, 64, 257), (2, 65, 30),
    (5, 70, 130), (1, 257, 1000), (2, 300, 20), (3, 513, 66), (1, 1500, 12), (2, 2049, 1), (600, 40, 3), (130, 17, 260),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", CASES)
def test_sequences_match_the_recurrence(case, dtype):
    B, T, F = case
    for k, (packed, done, ragged, carry) in enumerate(((False, 0.0, False, True), (True, 0.1, True, False), (True, 0.02, False, True))):
        ops = problem(sum(case) + k, B, T, F, dtype, packed, done, ragged, carry)
        cots = cotangents(k, B, T, F, dtype)
        outs, grads = run(ops, cots)
        assert outs[0].dtype == F32 and outs[1].dtype == dtype
        check(ops, cots, outs, grads)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(gated_scan(*ops.values()), outs))


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("F", [1, 2, 3, 4, 5, 17, 130, 1027])
def test_short_sequences(T, F):
    """Many of few steps: every form of them, with resets and sequences of no steps, and without a carry."""
    for B, dtype, packed, ragged, carry in ((70, F32, True, True, True), (301, BF16, False, False, False)):
        ops = problem(F * 8 + T, B, T, F, dtype, packed, 0.3, ragged, carry)
        cots = cotangents(F, B, T, F, dtype)
        outs, grads = run(ops, cots)
        check(ops, cots, outs, grads)
        again = run(ops, cots)
        assert all(torch.equal(a, b) for a, b in zip((*outs, *grads.values()), (*again[0], *again[1].values())))
        with torch.no_grad():
            alone = gated_scan(*(ops[n] for n in NAMES), ops["done"], ops["lengths"])
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))


@pytest.mark.parametrize("case", [(1, 9000, 16), (1, 2100, 520), (3, 3000, 40), (2, 8191, 3), (1, 4200, 100)])
def test_long_sequences_in_segments(case):
    B, T, F = case
    for dtype, ragged in ((F32, False), (BF16, True)):
        ops = problem(T, B, T, F, dtype, True, 0.001, ragged)
        cots = cotangents(T, B, T, F, dtype)
        outs, grads = run(ops, cots)
        check(ops, cots, outs, grads)


def test_steps_follow_the_sequence():
    for F, dtype in ((6, F32), (1, F32), (258, BF16)):
        ops = problem(F, 5, 12, F, dtype, True, 0.2)
        final, out = gated_scan(*ops.values())
        carry = ops["carry"].clone()
        for t in range(12):
            where = carry if t % 2 else None
            new, o = gated_scan_step(*(ops[n][:, t] for n in NAMES[:3]), ops["rate"], carry, ops["done"][:, t], out_carry=where)
            assert (new is carry) == (where is not None)
            carry = new
            torch.testing.assert_close(o, out[:, t], rtol=2 ** -7 if dtype == BF16 else 1e-5, atol=1e-5)
        torch.testing.assert_close(carry, final, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("F", [1, 3, 5, 64, 1003])
def test_one_step_in_place_and_apart(F):
    ops = problem(F, 9, 1, F, BF16)
    args = [ops[n][:, 0] for n in NAMES[:3]]
    done = torch.arange(9, device="cuda") % 3 == 0
    want, o = gated_scan_step(*args, ops["rate"], ops["carry"], done)
    final, out = gated_scan(*(ops[n] for n in NAMES), done[:, None])
    torch.testing.assert_close(want, final, rtol=1e-6, atol=1e-6)
    held = ops["carry"].clone()
    got, o2 = gated_scan_step(*args, ops["rate"], held, done, out_carry=held)
    assert got is held and torch.equal(got, want) and torch.equal(o, o2)


def test_one_used_output_and_some_gradients():
    ops = problem(3, 2, 70, 40, F32, done=0.05)
    cots = cotangents(1, 2, 70, 40, F32)
    for used in (0, 1):
        leaves = {n: ops[n].detach().requires_grad_() for n in NAMES}
        outs = gated_scan(*leaves.values(), ops["done"])
        grads = torch.autograd.grad(outs[used], list(leaves.values()), cots[used])
        check(ops, [c if k == used else None for k, c in enumerate(cots)], outs, dict(zip(NAMES, grads)))
    _, want = run(ops, cots)
    for name in NAMES:
        leaves = {n: ops[n].detach().requires_grad_(n == name) for n in NAMES}
        got, = torch.autograd.grad(gated_scan(*leaves.values(), ops["done"]), leaves[name], cots)
        assert torch.equal(got, want[name])


def test_small_and_large_decays():
    """Gates that shut or open fully, rates near 0 and far above 1: w from its series, states of one step."""
    gen = torch.Generator().manual_seed(4)
    B, T, F = 2, 50, 24
    x, i, d = (torch.randn(B, T, F, generator=gen).cuda() for _ in range(3))
    d[..., ::3] = -8.0
    d[..., 1::3] = 8.0
    rate = torch.tensor([1e-6, 1e-3, 0.1, 0.125, 0.13, 30.0]).repeat(4).cuda()
    ops = dict(x=x, input_gate=i, decay_gate=d, rate=rate, carry=torch.randn(B, F, generator=gen).cuda(), done=None, lengths=None)
    cots = cotangents(2, B, T, F, F32)
    outs, grads = run(ops, cots)
    check(ops, cots, outs, grads)
    ops["rate"] = torch.zeros(F, device="cuda")   # the state is kept, and no gradient is infinite
    outs, grads = run(ops, cots)
    assert torch.equal(outs[0], ops["carry"]) and all(torch.isfinite(v).all() for v in grads.values())


def test_decays_whose_input_weight_vanishes():
    """Gates of -60 to -100 and rates down to 1e-6: q = rate r runs from 1e-26 through the subnormal numbers to
    nothing.  The state stays the carry (w is at most sqrt(2 q) = 1.4e-13 a step), its gradient the sum of the cotangents; what
    reaches x and the gates is below |D| sqrt(2 q), and the rate below |D| |x| r / w = |D| |x| sqrt(r / (2 rate)) < 1e-9."""
    B, T, F = 2, 20, 64
    ops = problem(17, B, T, F, F32)
    ops["decay_gate"] = torch.linspace(-60, -100, F).repeat(B, T, 1).cuda()
    ops["rate"] = torch.logspace(0, -6, 7).repeat(10)[:F].cuda()
    cots = cotangents(18, B, T, F, F32)
    outs, grads = run(ops, cots)
    carry, dfinal, dout = np64(ops["carry"]), np64(cots[0]), np64(cots[1])
    within(outs[0], carry, T * 4 * N * np.abs(carry) + 1e-11)
    within(outs[1], np.broadcast_to(carry[:, None], (B, T, F)), T * 4 * N * np.abs(carry)[:, None] + 1e-11)
    within(grads["carry"], dfinal + dout.sum(1), 2 * T * N * (np.abs(dfinal) + np.abs(dout).sum(1)))
    for n in ("x", "input_gate", "decay_gate", "rate"):
        within(grads[n], np.zeros(grads[n].shape), 1e-8)


@pytest.mark.parametrize("T", [60, 3000])
def test_bad_steps_reach_what_follows_and_stop_at_a_reset(T):
    for bad in (float("nan"), float("inf")):
        for n in NAMES[:3]:
            ops = problem(5, 2, T, 24, BF16)
            ops["done"] = torch.zeros(2, T, dtype=torch.bool, device="cuda")
            ops["done"][:, T // 2] = True
            cots = cotangents(5, 2, T, 24, BF16)
            want_outs, want = run(ops, cots)
            ops[n][1, 7, 5] = bad
            outs, grads = run(ops, cots)
            # before the step, after the reset, in the other features and sequences: as they were
            touched = torch.zeros(2, T, 24, dtype=torch.bool, device="cuda")
            touched[1, 7:T // 2, 5] = True
            assert torch.equal(outs[1][~touched], want_outs[1][~touched]) and torch.equal(outs[0], want_outs[0])
            if bad != bad or n == "x":
                assert not torch.isfinite(outs[1][1, 7, 5])
            touched[1, :T // 2, 5] = True     # (gradients: back to the sequence's start)
            for k in NAMES[:3]:
                assert torch.equal(grads[k][~touched], want[k][~touched])


def test_rows_past_a_sequence_are_not_read():
    ops = problem(6, 3, 200, 40, BF16, ragged=True, done=0.05)
    ops["lengths"] = torch.tensor([200, 0, 77], dtype=torch.int32, device="cuda")
    cots = cotangents(6, 3, 200, 40, BF16)
    want_outs, want = run(ops, cots)
    past = torch.arange(200, device="cuda") >= ops["lengths"][:, None]
    for n in NAMES[:3]:
        ops[n][past] = float("nan")
    cots[1][past] = float("nan")
    ops["done"] |= past
    outs, grads = run(ops, cots)
    assert all(torch.equal(a, b) for a, b in zip((*outs, *grads.values()), (*want_outs, *want.values())))
    assert not outs[1][past].any() and not any(grads[n][past].any() for n in NAMES[:3])
    assert torch.equal(outs[0][1], ops["carry"][1]) and torch.equal(grads["carry"][1], cots[0][1])


def test_empty_batches_and_sequences():
    for B, T, F in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        ops = problem(7, B, T, F, F32)
        outs, grads = run(ops, cotangents(7, B, T, F, F32))
        assert outs[1].shape == (B, T, F) and outs[0].shape == (B, F) and not grads["rate"].any()
        if T == 0:
            assert torch.equal(outs[0], ops["carry"]) and grads["carry"].shape == (B, F)


def test_columns_and_cotangents_of_any_layout():
    ops = problem(8, 2, 40, 12, F32)
    cots = cotangents(8, 2, 40, 12, F32)
    want_outs, want = run(ops, cots)
    for n in NAMES[:3]:
        ops[n] = ops[n].transpose(1, 2).contiguous().transpose(1, 2)
    outs, grads = run(ops, [cots[0].t().contiguous().t(), cots[1].transpose(1, 2).contiguous().transpose(1, 2)])
    assert all(torch.equal(a, b) for a, b in zip((*outs, *grads.values()), (*want_outs, *want.values())))
    # one gate for all sequences: its gradient is their sum
    leaf = ops["decay_gate"][:1].clone().requires_grad_()
    got, = torch.autograd.grad(gated_scan(ops["x"], ops["input_gate"], leaf.expand(2, 40, 12), ops["rate"], ops["carry"]), leaf, cots)
    apart = dict(ops, decay_gate=leaf.detach().expand(2, 40, 12).contiguous())
    torch.testing.assert_close(got, run(apart, cots)[1]["decay_gate"].sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_the_same_twice():
    ops = problem(9, 700, 100, 70, BF16, True, 0.02)
    cots = cotangents(9, 700, 100, 70, BF16)
    a, b = run(ops, cots), run(ops, cots)
    assert all(torch.equal(x, y) for x, y in zip((*a[0], *a[1].values()), (*b[0], *b[1].values())))
    check(ops, cots, *a)


@pytest.mark.parametrize("size", [(2, 50, 32), (1, 3000, 24), (400, 3, 24), (5000, 8, 130)])
def test_a_captured_pass_replays(size):
    sets = [problem(10 + k, *size, BF16, done=0.05) for k in range(3)]
    cots = cotangents(1, *size, BF16)
    want = []
    for ops in sets:
        outs, grads = run(ops, cots)
        want.append([x.detach().clone() for x in (*outs, *grads.values())])
        del outs, grads
    leaves = {n: sets[0][n].clone().requires_grad_() for n in NAMES}
    done = sets[0]["done"].clone()

    def both():
        outs = gated_scan(*leaves.values(), done)
        return (*outs, *torch.autograd.grad(outs, list(leaves.values()), cots))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for k in (1, 2, 0, 1):
        with torch.no_grad():
            for n, x in leaves.items():
                x.copy_(sets[k][n])
            done.copy_(sets[k]["done"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def test_two_streams_at_once():
    sets = [problem(20 + k, 1, 9000, 48, F32, done=0.01) for k in range(2)]
    want = [gated_scan(*ops.values()) for ops in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for ops, stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            got.append(gated_scan(*ops.values()))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_steps_far_apart():
    """Operands wider than 2^23 elements a step are copied, those up to it read where they are, at 64-bit offsets."""
    for st in ((1 << 23) + 64, 1 << 23):
        T = 5 if st > 1 << 23 else 300
        wide = torch.zeros((T - 1) * st + 64, dtype=BF16, device="cuda")
        near = problem(11, 1, T, 16, BF16)
        x = wide.as_strided((1, T, 16), (0, st, 1))
        x.copy_(near["x"])
        cots = cotangents(11, 1, T, 16, BF16)
        a, b = run(near, cots), run(dict(near, x=x), cots)
        assert all(torch.equal(u, v) for u, v in zip((*a[0], *a[1].values()), (*b[0], *b[1].values())))
        del wide, x

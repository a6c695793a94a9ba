"""Linear attention with a decay for each head (chunked forward and backward,
and the step) against the float64 oracle (oracle/attention.py).

Tolerances, per element, from the oracle on absolute values (A: the sum of the
absolute values of the terms of that element):
- float32 arithmetic: a term passes through at most K + V + 2 C + T / C
  roundings of its product and sums (C >= 32 steps a chunk) and the powers of
  the decay, each within 2 ulp plus the exponent's rounding, T |g| / 2^23 in
  all; ROUNDS counts them, times 2^-24 A.
- bf16 storage: one rounding of the pair products and one of the state that
  enters a product, each 2^-8 of its terms, and the output's own, 2^-8 of its value;
  states and their cotangents stay float32.
- heads that share a key head are summed in float32 before the rounding.
"""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import linear_attention, linear_attention_step, qk_norm_rotary, rotary_frequencies
from oracle import attention as oat

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def np64(x):
    return None if x is None else x.detach().double().cpu().numpy()


def flags(x):
    return None if x is None else x.cpu().numpy()


def within(got, want, terms, dtype, rounds, name):
    got, want, terms = np64(got), np.asarray(want), np.asarray(terms)
    assert got.shape == want.shape, name
    tol = rounds * 2.0 ** -24 * terms + 1e-30
    if dtype == BF16:
        tol = tol + 2.0 ** -8 * (terms * 1.01 + np.abs(want))
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{name}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / tol):.3g} of "
                           f"the tolerance, first at {np.argwhere(bad)[0]}")


def problem(seed, B, T, H, G, K, V, dtype, done=0.0, ragged=False, carry=True, packed=False, slow=False):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen)

    if packed:
        whole = rand(B, T, H * K + G * (K + V) + 3).to(dtype).cuda()
        q = whole[..., 1:1 + H * K].unflatten(-1, (H, K))
        k = whole[..., 1 + H * K:1 + (H + G) * K].unflatten(-1, (G, K))
        v = whole[..., 1 + (H + G) * K:1 + (H + G) * K + G * V].unflatten(-1, (G, V))
    else:
        q, k, v = (rand(B, T, h, d).to(dtype).cuda() for h, d in ((H, K), (G, K), (G, V)))
    g = -(torch.rand(H, generator=gen) * (0.01 if slow else 0.3))
    g[0] = 0.0
    c = rand(B, H, K, V).cuda() if carry else None
    d = (torch.rand(B, T, generator=gen) < done).cuda() if done else None
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32)
        lengths[-1] = T
        lengths = lengths.cuda()
    return q, k, v, g.cuda(), c, d, lengths


def rounds_of(q, v, g):
    T, K, V = q.shape[1], q.shape[-1], v.shape[-1]
    return K + V + 128 + T // 32 + 20 + 2 * T * float(g.abs().max())


def check(q, k, v, g, carry, done, lengths, seed=0, scale=None):
    """Forward and gradients against the oracle."""
    dtype, (B, T, H, K), V = q.dtype, q.shape, v.shape[-1]
    gen = torch.Generator().manual_seed(seed + 77)
    leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, v, carry)]
    final, out = linear_attention(*leaves[:3], g, carry=leaves[3], done=done, lengths=lengths, scale=scale)
    assert final.dtype == F32 and out.dtype == dtype
    s = K ** -0.5 if scale is None else scale
    n = [np64(x) for x in (q, k, v, g, carry)]
    ops = (*n, flags(done), flags(lengths))
    absolute = [None if x is None else np.abs(x) for x in (*n[:3], n[4])]
    ops_abs = (*absolute[:3], n[3], absolute[3], flags(done), flags(lengths))
    rounds = rounds_of(q, v, g)
    want, terms = oat.linear_attention(*ops, s), oat.linear_attention(*ops_abs, abs(s))
    within(final, want[0], terms[0], F32, rounds, "final")
    within(out, want[1], terms[1], dtype, rounds, "out")
    dout = torch.randn(B, T, H, V, generator=gen).to(dtype).cuda()
    dfinal = torch.randn(B, H, K, V, generator=gen).cuda()
    grads = torch.autograd.grad([out, final], [x for x in leaves if x is not None], [dout, dfinal])
    want = oat.linear_attention_vjp(*ops, s, np64(dfinal), np64(dout))
    terms = oat.linear_attention_vjp(*ops_abs, abs(s), np.abs(np64(dfinal)), np.abs(np64(dout)))
    for i, got in enumerate(grads):
        within(got, want[i], terms[i], F32 if i == 3 else dtype, rounds, ("dq", "dk", "dv", "dcarry")[i])
    return final.detach(), out.detach(), grads


SHAPES = [  # batch, steps, heads, key heads, widths
    (1, 1, 1, 1, 1, 1), (2, 3, 2, 1, 5, 7), (1, 15, 3, 3, 16, 16), (2, 31, 2, 2, 32, 32), (1, 33, 2, 2, 33, 20),
    (2, 64, 4, 4, 64, 64), (1, 65, 4, 2, 64, 48), (3, 127, 2, 2, 8, 64), (1, 130, 2, 1, 128, 128), (2, 70, 1, 1, 100, 77),
    (2, 200, 6, 2, 24, 40), (2, 150, 2, 1, 96, 96), (1, 90, 3, 3, 80, 65),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequences_match_the_recurrence(shape, dtype):
    seed = sum(shape)
    check(*problem(seed, *shape, dtype), seed=seed)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(3, 3, 2, 1, 5, 7), (5, 70, 2, 2, 32, 32), (3, 150, 4, 2, 64, 64), (2, 130, 1, 1, 128, 96)])
@pytest.mark.parametrize("done,ragged,carry,packed", [(0.05, False, True, False), (0.0, True, True, True),
                                                      (0.1, True, False, True), (0.9, True, True, False)])
def test_resets_lengths_and_strides(shape, done, ragged, carry, packed, dtype):
    seed = sum(shape) + int(100 * done)
    check(*problem(seed, *shape, dtype, done=done, ragged=ragged, carry=carry, packed=packed), seed=seed)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,done,ragged", [((1, 1100, 1, 1, 24, 40), 0.0, False), ((2, 1300, 2, 1, 64, 64), 0.002, True),
                                               ((1, 1500, 1, 1, 128, 128), 0.001, False),
                                               ((2, 1100, 2, 2, 96, 72), 0.002, True)])
def test_long_sequences_are_cut_into_segments(shape, done, ragged, dtype):
    ops = problem(sum(shape), *shape, dtype, done=done, ragged=ragged, slow=True)
    check(*ops, seed=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1100, 2, 1, 64, 64), (2, 1200, 1, 1, 128, 128)])
def test_long_sequences_without_a_carry(shape, dtype):
    """Nothing asks for the backward's own states: their terms are kept shorter."""
    check(*problem(sum(shape), *shape, dtype, done=0.001, carry=False, slow=True), seed=2)


def test_lengths_of_zero_leave_the_carry():
    q, k, v, g, carry, _, _ = problem(5, 2, 40, 2, 2, 16, 16, F32)
    lengths = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    final, out, grads = check(q, k, v, g, carry, None, lengths)
    assert torch.equal(final[0], carry[0]) and not out[0].any()
    assert not any(x[0].any() for x in grads[:3])
    for T, B in ((0, 2), (3, 0)):
        q, k, v, g, carry, _, _ = problem(6, B, T, 2, 1, 16, 8, BF16)
        leaves = [x.requires_grad_() for x in (q, k, v, carry)]
        final, out = linear_attention(*leaves[:3], g, carry=leaves[3])
        assert out.shape == (B, T, 2, 8) and torch.equal(final, carry)
        grads = torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)])
        assert all(x.shape == y.shape for x, y in zip(grads, leaves)) and torch.equal(grads[3], torch.ones_like(carry))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_past_a_length_are_not_read(dtype):
    q, k, v, g, carry, done, _ = problem(7, 3, 100, 2, 1, 64, 64, dtype, done=0.05)
    lengths = torch.tensor([70, 0, 33], dtype=torch.int32, device="cuda")
    past = torch.arange(100, device="cuda") >= lengths[:, None]
    want = check(q, k, v, g, carry, done, lengths)
    for x in (q, k, v):
        x[past] = float("nan")
    done[past] = True
    got = check_raw(q, k, v, g, carry, done, lengths)
    for a, b in zip((want[0], want[1], *want[2]), got):
        assert torch.equal(a, b)


def check_raw(q, k, v, g, carry, done, lengths):
    gen = torch.Generator().manual_seed(77)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, carry)]
    final, out = linear_attention(*leaves[:3], g, carry=leaves[3], done=done, lengths=lengths)
    dout = torch.randn(out.shape, generator=gen).to(q.dtype).cuda()
    dfinal = torch.randn(final.shape, generator=gen).cuda()
    return (final.detach(), out.detach(), *torch.autograd.grad([out, final], leaves, [dout, dfinal]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("where", ["q", "k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_step_reaches_its_own_future_only(where, bad, dtype):
    """Steps before it and the next episode are as without it."""
    q, k, v, g, carry, _, _ = problem(8, 1, 160, 2, 2, 40, 40, dtype)
    done = torch.zeros(1, 160, dtype=torch.bool, device="cuda")
    done[0, 100] = True
    clean_final, clean, _ = check(q, k, v, g, carry, done, None)
    x = {"q": q, "k": k, "v": v}[where]
    x[0, 75, 1, 3] = bad
    final, out = linear_attention(q, k, v, g, carry=carry, done=done)
    assert torch.isfinite(final).all() and torch.isfinite(out[:, :75]).all() and torch.isfinite(out[:, 100:]).all()
    assert torch.equal(out[:, :, 0], clean[:, :, 0])
    n = [np64(y) for y in (q, k, v, g, carry)]
    with np.errstate(invalid="ignore"):
        want = oat.linear_attention(*n, flags(done), None, 40 ** -0.5)
    assert (np.isfinite(np64(out)) == np.isfinite(want[1])).all()
    terms = oat.linear_attention(*[np.abs(np.nan_to_num(y, posinf=0.0)) for y in n[:3]], n[3], np.abs(n[4]), flags(done),
                                 None, 40 ** -0.5)
    fine = np.isfinite(want[1])
    rounds = rounds_of(q, v, g)
    for got, w, t, dt in ((out, want[1], terms[1], dtype), (final, want[0], terms[0], F32)):
        f = np.isfinite(w)
        within(torch.nan_to_num(got.double(), posinf=0.0, neginf=0.0) * torch.from_numpy(f).cuda(),
               np.where(f, w, 0), t, dt, rounds, where)
    assert fine.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("reset", [None, 360, 700])
@pytest.mark.parametrize("bad", [0, 330, 355, 1299])
def test_a_bad_step_of_a_long_sequence(bad, reset, dtype):
    """In a segment whose state is formed from its end: finite where the recurrence is, forward and backward."""
    q, k, v, g, carry, _, _ = problem(17, 1, 1300, 1, 1, 33, 48, dtype, slow=True)
    done = torch.zeros(1, 1300, dtype=torch.bool, device="cuda")
    if reset is not None:
        done[0, reset] = True
    v[0, bad, 0, 7] = float("nan")
    got = check_raw(q, k, v, g, carry, done, None)
    n = [np64(x) for x in (q, k, v, g, carry)]
    gen = torch.Generator().manual_seed(77)
    dout = torch.randn(1, 1300, 1, 48, generator=gen).to(dtype).double().numpy()
    dfinal = torch.randn(1, 1, 33, 48, generator=gen).double().numpy()
    with np.errstate(invalid="ignore"):
        want = (*oat.linear_attention(*n, flags(done), None, 33 ** -0.5),
                *oat.linear_attention_vjp(*n, flags(done), None, 33 ** -0.5, dfinal, dout))
    for name, a, b in zip(("final", "out", "dq", "dk", "dv", "dcarry"), got, want):
        fine = np.isfinite(b)
        assert (np.isfinite(np64(a)) == fine).all(), name
        a = np64(a)[fine]
        assert np.linalg.norm(a - b[fine]) <= (1e-5 if dtype == F32 else 2 ** -7) * np.linalg.norm(b[fine]), name


def test_a_decay_of_zero_keeps_the_step_alone():
    q, k, v, _, carry, _, _ = problem(9, 1, 50, 2, 2, 16, 16, F32)
    g = torch.tensor([float("-inf"), -200.0], device="cuda")
    final, out = linear_attention(q, k, v, g, carry=carry, scale=1.0)
    n = [np64(x) for x in (q, k, v)]
    want = (n[0] * n[1]).sum(-1, keepdims=True) * n[2]
    within(out, want, (np.abs(n[0] * n[1])).sum(-1, keepdims=True) * np.abs(n[2]), F32, 200, "out")
    within(final, n[1][:, -1, :, :, None] * n[2][:, -1, :, None], np.abs(n[1][:, -1, :, :, None] * n[2][:, -1, :, None]),
           F32, 200, "final")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 20, 33), (5, 6, 3, 64, 64), (2, 2, 2, 128, 128), (70, 8, 4, 128, 48),
                                   (3, 2, 1, 77, 100)])
def test_a_step_is_a_sequence_of_one(shape, dtype):
    B, H, G, K, V = shape
    q, k, v, g, carry, done, _ = problem(sum(shape), B, 1, H, G, K, V, dtype, done=0.3, packed=True)
    got = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, carry, done=done[:, 0])
    n = [np64(x) for x in (q, k, v, g, carry)]
    want = oat.linear_attention(*n, flags(done), None, K ** -0.5)
    terms = oat.linear_attention(*map(np.abs, n[:3]), n[3], np.abs(n[4]), flags(done), None, K ** -0.5)
    within(got[0], want[0], terms[0], F32, 20, "carry")
    within(got[1][:, None], want[1], terms[1], F32 if dtype == F32 else BF16, K + 20, "out")
    kept = carry.clone()
    same, out = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, carry, done=done[:, 0], out_carry=carry)
    assert same is carry and torch.equal(carry, got[0]) and torch.equal(out, got[1]) and not torch.equal(kept, carry)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_after_norms_follow_the_sequence(dtype):
    """The three as a torso uses them: normed, turned queries and keys, a
    sequence with resets for the update, its steps one by one for the rollout."""
    B, T, H, G, D = 3, 70, 4, 2, 32
    q, k, v, g, carry, done, _ = problem(11, B, T, H, G, D, D, dtype, done=0.05, packed=True)
    gen = torch.Generator().manual_seed(12)
    scales = [(1 + 0.1 * torch.randn(D, generator=gen)).cuda() for _ in range(2)]
    f = rotary_frequencies(16)
    positions = (torch.arange(T, dtype=torch.int32) + torch.tensor([[5], [0], [9000]], dtype=torch.int32)).cuda()
    leaves = [x.detach().requires_grad_() for x in (q, k, v, carry, *scales)]
    nq, nk = qk_norm_rotary(leaves[0], leaves[1], leaves[4], leaves[5], f, positions)
    final, out = linear_attention(nq, nk, leaves[2], g, carry=leaves[3], done=done)
    state, steps = carry, []
    for t in range(T):
        sq, sk = qk_norm_rotary(q[:, t:t + 1], k[:, t:t + 1], *scales, f, positions[:, t:t + 1])
        assert torch.equal(sq, nq[:, t:t + 1]) and torch.equal(sk, nk[:, t:t + 1])
        state, o = linear_attention_step(sq[:, 0], sk[:, 0], v[:, t], g, state, done=done[:, t])
        steps.append(o)
    pq, pk = np64(nq), np64(nk)
    ops = (pq, pk, np64(v), np64(g), np64(carry), flags(done), None)
    terms = oat.linear_attention(np.abs(pq), np.abs(pk), np.abs(np64(v)), np64(g), np.abs(np64(carry)), flags(done), None,
                                 D ** -0.5)
    want = oat.linear_attention(*ops, D ** -0.5)
    for got in ((final, out), (state, torch.stack(steps, 1))):
        within(got[0], want[0], terms[0], F32, rounds_of(q, v, g), "final")
        within(got[1], want[1], terms[1], dtype, rounds_of(q, v, g), "out")
    # gradients through both against the oracle's chain, in the norm
    dout, dfinal = torch.randn(out.shape, generator=gen).to(dtype).cuda(), torch.randn(final.shape, generator=gen).cuda()
    grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    s = [np64(x) for x in scales]
    nq64, nk64 = (oat.norm_rotary(np64(x), w, np64(f), flags(positions), 1e-6) for x, w in ((q, s[0]), (k, s[1])))
    dq, dk, dv, dc = oat.linear_attention_vjp(nq64, nk64, *ops[2:], D ** -0.5, np64(dfinal), np64(dout))
    chain = [oat.norm_rotary_vjp(np64(x), w, np64(f), flags(positions), 1e-6, False, c)
             for x, w, c in ((q, s[0], dq), (k, s[1], dk))]
    # bf16: at most five roundings of 2^-8 in a row (normed operands, pairs or state, cotangent, gradient), in the norm
    bound = 1e-5 if dtype == F32 else 5 * 2.0 ** -8
    for got, w in zip(grads, (chain[0][0], chain[1][0], dv, dc, chain[0][1], chain[1][1])):
        assert np.linalg.norm(np64(got) - w) <= bound * np.linalg.norm(w)


def test_only_the_final_carry_or_only_the_outputs():
    q, k, v, g, carry, _, _ = problem(13, 2, 40, 2, 1, 16, 24, F32)
    n = [np64(x) for x in (q, k, v, g, carry)]
    for which in (0, 1):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, carry)]
        result = linear_attention(*leaves[:3], g, carry=leaves[3])[which]
        cot = torch.randn(result.shape, generator=torch.Generator().manual_seed(3)).cuda()
        grads = torch.autograd.grad(result, leaves, cot)
        other = np.zeros((2, 40, 2, 24)) if which == 0 else None
        args = (np64(cot), other) if which == 0 else (None, np64(cot))
        want = oat.linear_attention_vjp(*n, None, None, 0.25, *args)
        for a, b in zip(grads, want):
            np.testing.assert_allclose(np64(a), b, rtol=0, atol=2e-5 * np.abs(b).max())


def test_shared_and_expanded_heads_agree():
    q, k, v, g, carry, done, _ = problem(14, 2, 90, 4, 1, 32, 32, F32, done=0.05)
    cot = torch.randn(2, 90, 4, 32, generator=torch.Generator().manual_seed(3)).cuda()
    got = []
    for expand in (False, True):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        kk, vv = (x.expand(-1, -1, 4, -1) if expand else x for x in leaves[1:])
        out = linear_attention(leaves[0], kk, vv, g, carry=carry, done=done)[1]
        got.append((out, *torch.autograd.grad(out, leaves, cot)))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    for a, b in zip(got[0][2:], got[1][2:]):
        assert a.shape == b.shape and (a - b).norm() <= 1e-6 * b.norm()


def test_orders_of_axes_and_the_same_twice():
    """Operands whose axes are in another order; two runs give the same bits."""
    q, k, v, g, carry, done, _ = problem(15, 3, 77, 2, 2, 48, 48, BF16, done=0.05)
    a = check_raw(q, k, v, g, carry, done, None)
    moved = [x.permute(2, 3, 0, 1).contiguous().permute(2, 3, 0, 1) for x in (q, k, v)]
    time_major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    for ops in ((q, k, v), moved, time_major):
        b = check_raw(*ops, g, carry, done, None)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_step_of_a_wide_time_major_batch():
    """Of one step the step's stride says nothing: here it is that of a whole
    batch, past what the kernels count in."""
    B, H, K = 66000, 16, 8
    gen = torch.Generator().manual_seed(17)
    ops = [torch.randn(1, B, H, K, generator=gen).to(BF16).cuda().transpose(0, 1).requires_grad_() for _ in range(3)]
    assert ops[0].stride(1) > 1 << 23
    g = torch.full((H,), -0.1).cuda()
    final, out = linear_attention(*ops, g)
    grads = torch.autograd.grad(out, ops, out.detach())
    q, k, v = (x.detach()[:, 0].float() for x in ops)
    w = (q * k).sum(-1, keepdim=True) * K ** -0.5
    # one product of at most K + 2 float32 roundings of 2^-24, the pair products rounded to bf16, and the outputs
    close = lambda a, b, terms: ((a[:, 0].float() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -7 * terms + 1e-30).all()
    assert close(out, w * v, (q * k).abs().sum(-1, keepdim=True) * K ** -0.5 * v.abs())
    assert torch.equal(final, k[..., None] * v[..., None, :])
    do = out.detach()[:, 0].float()
    assert close(grads[2], w * do, (q * k).abs().sum(-1, keepdim=True) * K ** -0.5 * do.abs())
    d = (do * v).sum(-1, keepdim=True) * K ** -0.5
    terms = (do * v).abs().sum(-1, keepdim=True) * K ** -0.5
    assert close(grads[0], d * k, terms * k.abs()) and close(grads[1], d * q, terms * q.abs())


def test_a_second_derivative_is_refused():
    q, k, v, g, _, _, _ = problem(16, 1, 5, 1, 1, 8, 8, F32)
    q.requires_grad_()
    out = linear_attention(q, k, v, g)[1]
    dq, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)


def test_captured_sequences_and_steps_replay():
    """A captured forward, backward and step, replayed with other inputs in
    place, between eager calls on another stream."""
    shape = (2, 700, 2, 1, 64, 64)
    sets = [problem(20 + i, *shape, BF16, done=0.01, slow=True) for i in range(3)]
    want = [check_raw(*s) for s in sets]
    steps = [linear_attention_step(*(x[:, 0] for x in s[:3]), s[3], s[4]) for s in sets]
    q, k, v, g, carry, done, _ = [None if x is None else x.clone() for x in sets[0]]
    gen = torch.Generator().manual_seed(77)
    dout = torch.randn(2, 700, 2, 64, generator=gen).to(BF16).cuda()
    dfinal = torch.randn(carry.shape, generator=gen).cuda()
    leaves = [x.requires_grad_() for x in (q, k, v, carry)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            final, out = linear_attention(q, k, v, g, carry=carry, done=done)
            torch.autograd.grad([out, final], leaves, [dout, dfinal])
            del final, out
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        final, out = linear_attention(q, k, v, g, carry=carry, done=done)
        grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
        with torch.no_grad():
            step = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, carry)
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            for x, y in zip((q, k, v, g, carry, done), sets[i]):
                x.copy_(y)
        graph.replay()
        with torch.cuda.stream(side):
            check_raw(*sets[i])
        for a, b in zip((final, out, *grads, *step), (*want[i], *steps[i])):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_work_on_another_stream():
    s = problem(30, 4, 300, 4, 4, 64, 64, BF16, done=0.01)
    want = check_raw(*s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = check_raw(*s)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(8192, 70, 2, 2, 20, 33), (12000, 69, 2, 2, 24, 32), (8192, 65, 2, 2, 64, 64),
                                   (4096, 70, 2, 2, 128, 120), (8192, 66, 2, 1, 40, 64)])
def test_large_batches_are_their_parts(shape, dtype):
    """Outputs large enough to be streamed, an infinity and a NaN among them: to
    the bit those of eighths of the batch, which are not."""
    _, T, H, G, K, V = shape
    B = shape[0] * 2 // dtype.itemsize
    assert B * T * H * V * dtype.itemsize >= 64 << 20
    assert B // 8 * T * H * (2 * K + V) * dtype.itemsize < 64 << 20
    gen = torch.Generator("cuda").manual_seed(sum(shape))
    q, k, v, dout = (torch.randn(B, T, h, d, generator=gen, device="cuda").to(dtype)
                     for h, d in ((H, K), (G, K), (G, V), (H, V)))
    q[5, 30, 0, 3], k[B // 2, 11, 0, 1], v[B - 1, T - 2, 0, 0] = float("inf"), float("nan"), float("-inf")
    carry = torch.randn(B, H, K, V, generator=gen, device="cuda")
    done = torch.rand(B, T, generator=gen, device="cuda") < 0.01
    lengths = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    lengths[[5, B // 2, B - 1]] = T
    g = torch.tensor([-0.01, -0.2], device="cuda")

    def both_passes(rows):
        leaves = [x[rows].requires_grad_() for x in (q, k, v, carry)]
        final, out = linear_attention(*leaves[:3], g, carry=leaves[3], done=done[rows], lengths=lengths[rows])
        return final.detach(), out.detach(), *torch.autograd.grad(out, leaves, dout[rows])

    whole = both_passes(slice(0, B))
    for i in range(8):
        rows = slice(i * B // 8, (i + 1) * B // 8)
        for a, b in zip(whole, both_passes(rows)):
            torch.testing.assert_close(a[rows], b, rtol=0, atol=0, equal_nan=True)


def test_two_graphs_and_two_streams_at_once():
    """Two captured passes, replayed at the same time, and two eager calls: each
    has its own workspace."""
    sets = [problem(40 + i, 2, 900, 2, 1, 64, 64, BF16, done=0.01, slow=True) for i in range(2)]
    gen = torch.Generator().manual_seed(5)
    dout = torch.randn(2, 900, 2, 64, generator=gen).to(BF16).cuda()
    dfinal = torch.randn(2, 2, 64, 64, generator=gen).cuda()

    def both_passes(q, k, v, g, carry, done, _):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, carry)]
        final, out = linear_attention(*leaves[:3], g, carry=leaves[3], done=done)
        return (final.detach(), out.detach(), *torch.autograd.grad([out, final], leaves, [dout, dfinal]))

    want = [both_passes(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, got = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(both_passes(*s))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        eager = []
        for stream, graph in zip(streams, graphs):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                eager.append(both_passes(*s))
        torch.cuda.synchronize()
        for results in (got, eager):
            for a, b in zip(results, want):
                assert all(torch.equal(x, y) for x, y in zip(a, b))

"""How near linear attention's sequences come to the float64 oracle
(oracle/attention.py), where every head's state decays: each element against
its roundings, and the norms of whole results.

Per element, A the sum of the absolute values of its terms (the oracle on
absolute values):
- float32 arithmetic as in test_gpu_linear_attention.py: rounds_of() roundings
  of 2^-24 A;
- bf16 storage: a term meets a pair product or an entering state, each in two
  bf16 pieces, which leave at most 2^-17 of it, and a state's own terms keep at
  least two: 2^-16 A in all.  The output is rounded once, 2^-8 of its value.
In the norm: a result with N independent roundings is off by sqrt(N / 3) 2^-24
of its norm, below 1e-6 for N up to 800 (K + V + 2 C + T / C here); an output
rounded to bf16 by at most 2^-8 / sqrt(3).
"""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import linear_attention, linear_attention_step
from oracle import attention as oat
from test_gpu_linear_attention import BF16, F32, flags, np64, problem, rounds_of

pytestmark = pytest.mark.gpu

NORM_F32, NORM_BF16 = 1e-6, 2.0 ** -8 / 3 ** 0.5


def decaying(seed, *shape_and_dtype, slow=False, **kw):
    q, k, v, g, *rest = problem(seed, *shape_and_dtype, slow=slow, **kw)
    g[0] = -0.003 if slow else -0.05
    return q, k, v, g, *rest


def near(got, want, terms, dtype, rounds, name):
    got = np64(got)
    tol = rounds * 2.0 ** -24 * terms + 1e-30
    if dtype == BF16:
        tol = tol + 2.0 ** -16 * terms
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    off = np.abs(got - want)
    assert (off <= tol).all(), f"{name}: {(off > tol).sum()} of {off.size} off, worst {np.max(off / tol):.3g}"
    norm = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    print(f"{name}: {norm:.3g} of the norm, worst {np.max(off / tol):.3g} of the tolerance")
    assert norm <= (NORM_F32 if dtype == F32 else NORM_BF16), f"{name}: {norm:.3g} of the norm"


def both_passes(q, k, v, g, carry, done, lengths, seed):
    gen = torch.Generator().manual_seed(seed)
    leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, v, carry)]
    final, out = linear_attention(*leaves[:3], g, carry=leaves[3], done=done, lengths=lengths)
    dout = torch.randn(out.shape, generator=gen).to(q.dtype).cuda()
    dfinal = torch.randn(final.shape, generator=gen).cuda()
    return (final, out, *torch.autograd.grad([out, final], [x for x in leaves if x is not None], [dout, dfinal])), dfinal, dout


def oracle_passes(ops, scale, dfinal, dout):
    return (*oat.linear_attention(*ops, scale), *oat.linear_attention_vjp(*ops, scale, dfinal, dout))


NAMES = ("final", "out", "dq", "dk", "dv", "dcarry")


def check(q, k, v, g, carry, done, lengths, seed=0):
    got, dfinal, dout = both_passes(q, k, v, g, carry, done, lengths, seed)
    n = [np64(x) for x in (q, k, v, g, carry)]
    absolute = [None if x is None else np.abs(x) for x in n]
    scale, rounds = q.shape[-1] ** -0.5, rounds_of(q, v, g)
    want = oracle_passes((*n, flags(done), flags(lengths)), scale, np64(dfinal), np64(dout))
    terms = oracle_passes((*absolute[:3], n[3], absolute[4], flags(done), flags(lengths)), scale, np.abs(np64(dfinal)),
                          np.abs(np64(dout)))
    for name, a, w, t in zip(NAMES, got, want, terms):
        near(a, w, t, F32 if name in ("final", "dcarry") else q.dtype, rounds, name)


SHAPES = [  # batch, steps, heads, key heads, widths
    (2, 31, 2, 2, 32, 32), (3, 127, 2, 2, 8, 64), (2, 64, 4, 4, 64, 64), (1, 65, 1, 1, 64, 48), (2, 70, 1, 1, 100, 77),
    (2, 200, 6, 2, 24, 40), (2, 150, 2, 1, 96, 96), (1, 90, 1, 1, 80, 65), (1, 130, 2, 1, 128, 128), (2, 100, 1, 1, 128, 120),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("done,ragged,carry", [(0.0, False, True), (0.03, True, True), (0.1, False, False)])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequences(shape, done, ragged, carry, dtype):
    check(*decaying(sum(shape), *shape, dtype, done=done, ragged=ragged, carry=carry), seed=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("done,ragged,carry", [(0.0, False, True), (0.002, True, True), (0.001, False, False)])
@pytest.mark.parametrize("shape", [(1, 1100, 1, 1, 24, 40), (1, 900, 2, 1, 32, 32), (2, 1300, 2, 1, 64, 64),
                                   (2, 1100, 2, 2, 96, 72), (1, 1500, 1, 1, 128, 128), (2, 700, 2, 1, 128, 128)])
def test_segments(shape, done, ragged, carry, dtype):
    check(*decaying(sum(shape), *shape, dtype, done=done, ragged=ragged, carry=carry, slow=True), seed=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [48, 128])
@pytest.mark.parametrize("reset", [None, 360, 700])
@pytest.mark.parametrize("bad", [0, 330, 1099])
def test_a_bad_step_under_decay(bad, reset, width, dtype):
    """In a segment whose state is formed from its end: finite where the recurrence is, and near it there."""
    q, k, v, g, carry, _, _ = decaying(18, 1, 1100, 1, 1, width, width, dtype, slow=True)
    done = torch.zeros(1, 1100, dtype=torch.bool, device="cuda")
    if reset is not None:
        done[0, reset] = True
    v[0, bad, 0, 7] = float("nan")
    got, dfinal, dout = both_passes(q, k, v, g, carry, done, None, 3)
    n = [np64(x) for x in (q, k, v, g, carry)]
    with np.errstate(invalid="ignore"):
        want = oracle_passes((*n, flags(done), None), width ** -0.5, np64(dfinal), np64(dout))
    absolute = [np.abs(np.nan_to_num(x)) for x in n]
    terms = oracle_passes((*absolute[:3], n[3], absolute[4], flags(done), None), width ** -0.5, np.abs(np64(dfinal)),
                          np.abs(np64(dout)))
    for name, a, w, t in zip(NAMES, got, want, terms):
        fine = np.isfinite(w)
        assert (np.isfinite(np64(a)) == fine).all(), name
        if fine.any():   # (of dq nothing is, where the first step is bad)
            near(a.detach().cpu()[torch.from_numpy(fine)], w[fine], t[fine], F32 if name in ("final", "dcarry") else dtype,
                 rounds_of(q, v, g), name)


@pytest.mark.parametrize("width", [32, 64, 128])
def test_a_rollout_and_its_sequence_agree_in_bf16(width):
    """The steps one by one hold everything in float32: the sequence's outputs
    are theirs but for roundings that fall to either side."""
    B, T, H = 2, 100, 2
    q, k, v, g, carry, done, _ = decaying(19, B, T, H, 1, width, width, BF16, done=0.03)
    final, out = linear_attention(q, k, v, g, carry=carry, done=done)
    state, steps = carry, []
    for t in range(T):
        state, o = linear_attention_step(q[:, t], k[:, t], v[:, t], g, state, done=done[:, t])
        steps.append(o)
    steps = torch.stack(steps, 1)
    # two bf16 pieces leave 2.6e-6 of a result in the norm, in a state's terms, the state and the pair products: 5e-6
    # together, and a border between two bf16 values, 2^-8 of them apart or more, lies between in 0.1 % of the elements
    # of that size; more often in small ones, of which a tenth of the size, with ten times the share, are 8 %
    assert (out != steps).float().mean() <= 0.02
    assert (final - state).norm() <= NORM_F32 * state.norm()

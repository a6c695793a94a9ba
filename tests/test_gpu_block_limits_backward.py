"""The gated recurrence at the most steps, features and states it takes and the norms around a block at the most rows,
both passes, against the formulas in float64 on the host: the rows, steps and features at both ends.

N = 2^-24.  States and cotangents of states follow the recurrence: a sum of terms of sizes S_t = a_t S_{t-1} + |b_t| is off
by e_t = a_t e_{t-1} + 2 N ((16 q_t + 4) a_t S_{t-1} + 56 |b_t|) where b = w i x is within 56 (w within 40 where 1 - a^2 is
a difference at 1/8), and 12 N S_t where maps are joined.  Gradients are products of these, within (100 + 32 q) N of the sizes
of their terms.  bf16 outputs add their rounding, 2^-8 of the value."""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import gated_scan, gated_scan_step, residual_norm
from oracle import gated as og

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
N = 2.0 ** -24


def host(t):
    return t.detach().double().cpu().numpy()


def near(got, want, tol):
    assert got.shape == want.shape
    assert (np.abs(host(got) - want) <= tol + (2.0 ** -8 * np.abs(want) if got.dtype == BF16 else 0) + 1e-37).all()


def check(parts, carry, dfinal, out, final, grads, dcarry, steps=slice(None)):
    """parts: x, both gates and dout [batch, steps, features], rate; out and grads: those of `steps`; final, dcarry or None."""
    x, i, d, dout, rate = (host(t) for t in parts)
    carry, dfinal = host(carry), host(dfinal)
    g = og.gates(x, i, d, rate)
    last, want, before = og.gated_scan(x, i, d, rate, carry)
    a, q, b = g["a"], g["q"], np.abs(g["w"] * g["i"] * x)
    e, S, entering, errors = np.zeros_like(carry), np.abs(carry), np.zeros_like(x), np.zeros_like(x)
    for t in range(x.shape[1]):
        entering[:, t] = e + 12 * N * S
        e = a[:, t] * e + 2 * N * ((16 * q[:, t] + 4) * a[:, t] * S + 56 * b[:, t])
        S = a[:, t] * S + b[:, t]
        errors[:, t] = e + 12 * N * S
    near(out, want[:, steps], errors[:, steps])
    if final is not None:
        near(final, last, e + 12 * N * S)
    v = og.gated_scan_vjp(x, i, d, rate, carry, None, None, dfinal, dout)
    eE, S, eD = np.zeros_like(carry), np.abs(dfinal), np.zeros_like(x)
    for t in range(x.shape[1] - 1, -1, -1):
        S = S + np.abs(dout[:, t])
        eD[:, t] = eE + 12 * N * S
        eE, S = a[:, t] * (eE + 2 * N * (16 * q[:, t] + 4) * S), a[:, t] * S
    D = np.abs(v["D"])
    size = (100 + 32 * q) * N * D + eD
    u = np.abs(g["i"] * x)
    slope = size * (np.abs(a * before) + a * a * u / g["w"]) + D * a * entering
    near(grads[0], v["x"][:, steps], (size * g["w"] * g["i"])[:, steps])
    near(grads[1], v["input_gate"][:, steps], (size * g["w"] * u * (1 - g["i"]))[:, steps])
    near(grads[2], v["decay_gate"][:, steps], (slope * q * (1 - g["r"]))[:, steps])
    if dcarry is not None:
        near(dcarry, v["carry"], eE + 12 * N * S)


def test_the_longest_sequence_and_its_gradients():
    """2^30 steps of one feature.  The decays of 2048 of them leave nothing (their exponents' mean is -1.5): the first
    and the last 2048 are those of the 4096 at either end."""
    T, near_steps = 1 << 30, 2048
    gen = torch.Generator(device="cuda").manual_seed(6)
    pieces = torch.randn(4, 1 << 22, generator=gen, device="cuda").to(BF16)
    x, i, d, dout = (p.repeat(T >> 22).view(1, T, 1) for p in pieces)
    rate, carry, dfinal = (torch.tensor(v, device="cuda") for v in ([3.0], [[7.0]], [[-2.0]]))
    leaves = [t.requires_grad_() for t in (x, i, d, carry)]
    final, out = gated_scan(*leaves[:3], rate, leaves[3])
    *grads, dcarry = torch.autograd.grad([final, out], leaves, [dfinal, dout])
    zero, both = torch.zeros(1, 1), 2 * near_steps
    first, last = (lambda t: t[:, :both]), (lambda t: t[:, -both:])
    whole = [x, i, d, dout]
    kept = slice(0, near_steps)
    check([*map(first, whole), rate], carry, zero, out[:, kept], None, [g[:, kept] for g in grads], dcarry, kept)
    kept = slice(-near_steps, None)
    check([*map(last, whole), rate], zero, dfinal, out[:, kept], final, [g[:, kept] for g in grads], None, kept)


@pytest.mark.parametrize("B,T", [(1, 40), (512, 2), (512, 9)])
def test_the_most_features_and_states(B, T):
    """2^20 features; of 512 sequences, 2^29 states.  Their ends, and where two workgroups' features meet."""
    F = 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(T)

    def normal(*shape, dtype=BF16):
        t = torch.empty(*shape, dtype=dtype, device="cuda")
        for b in range(shape[0]):
            t[b] = torch.randn(shape[1:], generator=gen, device="cuda").to(dtype)
        return t

    x, i, d, dout = (normal(B, T, F) for _ in range(4))
    carry, dfinal = (normal(B, F, dtype=F32) for _ in range(2))
    rate = torch.exp(torch.empty(F, device="cuda").uniform_(-4, 1, generator=gen))
    leaves = [t.requires_grad_() for t in (x, i, d, rate, carry)]
    final, out = gated_scan(*leaves)
    *grads, drate, dcarry = torch.autograd.grad([final, out], leaves, [dfinal, dout])
    step, first = gated_scan_step(*(t.detach()[:, 0] for t in leaves[:3]), rate.detach(), carry.detach())
    rows = torch.tensor(sorted({0, B // 2, B - 1}), device="cuda")
    for f in (slice(0, 300), slice(F // 2 - 150, F // 2 + 150), slice(F - 300, F)):
        def some(t):
            return t.detach()[rows][..., f]
        check([*map(some, (x, i, d, dout)), rate[f]], some(carry), some(dfinal), some(out), some(final), [some(g) for g in grads],
              some(dcarry))
        want = og.gated_scan(*(host(some(t))[:, :1] for t in (x, i, d)), host(rate[f]), host(some(carry)))[0]
        q = og.gates(*(host(some(t))[:, 0] for t in (x, i, d)), host(rate[f]))
        tol = 2 * N * ((16 * q["q"] + 16) * q["a"] * np.abs(host(some(carry))) + 68 * np.abs(q["w"] * q["i"] * host(some(x))[:, 0]))
        near(some(step), want, tol)
        near(some(first), want, tol)
        # the rate's: all sequences of a few features
        columns = slice(f.start, f.start + 3)
        some_d = [host(t.detach()[..., columns]) for t in (x, i, d, rate, carry, dfinal, dout)]
        v = og.gated_scan_vjp(*some_d[:5], None, None, *some_d[5:])
        g = og.gates(*some_d[:4])
        _, _, before = og.gated_scan(*some_d[:5])
        S = np.abs(some_d[5]) + np.abs(some_d[6]).sum(1)
        terms = S[:, None] * (np.abs(g["a"]) * (np.abs(some_d[4]) + np.abs(g["w"] * g["i"] * some_d[0]).sum(1))[:, None]
                              + g["a"] ** 2 * np.abs(g["i"] * some_d[0]) / g["w"]) * g["r"]
        near(drate[columns], v["rate"], (T / 8 + B + 300) * N * terms.sum((0, 1)))


def test_the_most_rows_between_blocks_and_their_gradients():
    """2^31 - 2^20 - 1 rows of one column: n = u ru, y = x + s n, z = y ry p with ru = 1 / sqrt(u^2 + eps).  One column's
    norms keep hardly more than the sign: their slopes are eps ru^3 and eps ry^3, differences of numbers near 1 that the
    kernel forms as such, off by 60 roundings of ru and ry, 1 / sqrt(eps) = 1000 each at most.  y is off by 8 N (|x| + 1), and ry,
    which goes as 1 / y, by that over |y| and 20 more."""
    rows, ends, eps = (1 << 31) - (1 << 20) - 1, 1 << 14, 1e-6
    gen = torch.Generator(device="cuda").manual_seed(3)
    u, x, dy, dz = torch.randn(4, ends, generator=gen, device="cuda").to(BF16)
    block, residual, dstream, dnormed = (torch.zeros(1, rows, 1, dtype=BF16, device="cuda") for _ in range(4))
    for whole, part in ((block, u), (residual, x), (dstream, dy), (dnormed, dz)):
        whole[0, :ends, 0], whole[0, -ends:, 0] = part, part.flip(0)
    scale, pre = (torch.tensor([v], device="cuda").requires_grad_() for v in (1.25, 0.75))
    leaves = [block.requires_grad_(), residual.requires_grad_(), scale, pre]
    outs = residual_norm(block, residual, residual_scale=scale, pre_scale=pre, epsilon=eps)
    dblock, dresidual, dscale, dpre = torch.autograd.grad(outs, leaves, [dstream, dnormed])
    u, x, dy, dz = (t.double() for t in (u, x, dy, dz))
    ru = (u * u + eps).rsqrt()
    n = u * ru
    y = x + 1.25 * n
    ry = (y * y + eps).rsqrt()
    dx = dy + dz * 0.75 * eps * ry ** 3
    du = dx * 1.25 * eps * ru ** 3
    off = 60 + 8 * (x.abs() + 2) / (y.abs() + 1e-3)      # roundings of ry, and of y ry
    dx_off = 4 * N * dy.abs() + 4 * off * N * ry * (0.75 * dz.abs())
    du_off = 1.25 * ru * (200 * N * (dy.abs() + 0.75 * dz.abs() * ry) + 2 * dx_off)
    for got, want, tol in ((outs[0], y, 8 * N * (x.abs() + 2)), (outs[1], 0.75 * y * ry, off * N), (dresidual, dx, dx_off),
                           (dblock, du, du_off)):
        for end in (got.detach()[0, :ends, 0], got.detach()[0, -ends:, 0].flip(0)):
            assert ((end.double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()
        assert not got.detach()[0, ends:rows - ends:9973].any()
    terms = 2 * (dy.abs() + 0.75 * dz.abs() * ry) * n.abs()
    assert abs(dscale.item() - 2 * (dx * n).sum().item()) <= (ends * N * terms + 2 * dx_off).sum().item()
    assert abs(dpre.item() - 2 * (dz * y * ry).sum().item()) <= (2 * dz.abs() * (off + ends) * N).sum().item()

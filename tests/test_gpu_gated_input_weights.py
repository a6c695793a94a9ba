"""The gated recurrence's input weights w = sqrt(1 - a^2) over all decays, and densely about 2 rate r = 1/8, where the
kernels go from a series to the difference: every step starts an episode, so that an output is w i x alone and a
gradient that of its own step.

Tolerances, in roundings N = 2^-24, with q = rate r.  A sigmoid is within 12, what it leaves of 1 within 16 (arguments up
to 8: an exponent of 11.5 off by a rounding and its constant's), q within 16 of its value and a within A = 16 q + 4 of its.  Below 2 q = 1/8 the series is within 20 of 1 - a^2: 16 of
q's, its polynomial 3, a product.  Above, the difference is off by twice a's error, 2 A a^2 / (1 - a^2), and its own
rounding: 76 at the switch, where a^2 = 0.88, and less above.  So w is within W = half of that and 2 for the root:
40 at the switch.  An output takes w, i and two products: W + 15; dx the same and a product; dinput_gate W + 12 + 16 + 5.
ddecay_gate = D a^2 i x / w rate r (1 - r) takes W, 2 A, the sigmoids' 40 and 9 products: W + 2 A + 49; past the type's normal
range 1e-37."""
import math

import pytest
import torch

from boonta_amd.kernels import gated_scan, gated_scan_step

pytestmark = pytest.mark.gpu

N = 2.0 ** -24


def rates():
    """q where the decay gate is 8 (r = 0.99966): 3000 about 1/16, and from 1e-6 to 30."""
    about = torch.linspace(0.0620, 0.0631, 3000)
    wide = torch.logspace(-6, math.log10(30.0), 1024)
    return torch.cat([about, wide])


@pytest.mark.parametrize("T", [1, 4, 8, 40])
def test_outputs_and_gradients_of_single_steps(T):
    gen = torch.Generator().manual_seed(T)
    rate = rates().cuda()
    F, B = rate.numel(), 3
    x, i = (torch.randn(B, T, F, generator=gen).cuda() for _ in range(2))
    # about 8, and (the last sequence) 0 for twice the rate
    d = torch.full((B, T, F), 8.0, device="cuda")
    d[-1] = 0.0
    d += 1e-3 * torch.randn(B, T, F, generator=gen).cuda()
    scale = torch.where(torch.arange(F, device="cuda") % 2 == 0, 1.0, 2.0)
    rate = rate * scale                       # (of r = 1/2 the odd ones are about the switch)
    done = torch.ones(B, T, dtype=torch.bool, device="cuda")
    leaves = [t.requires_grad_() for t in (x, i, d)]
    _, out = gated_scan(*leaves, rate, None, done)
    dout = torch.randn(B, T, F, generator=gen).cuda()
    dx, di, dd = torch.autograd.grad(out, leaves, dout)

    X, I, D, R, G = (t.detach().double() for t in (x, i, d, rate, dout))
    si, sd = torch.sigmoid(I), torch.sigmoid(D)
    q = R * sd
    w2, a2 = -torch.expm1(-2 * q), torch.exp(-2 * q)
    w, A = torch.sqrt(w2), 16 * q + 4
    # (either form at the switch itself)
    series, difference = torch.full_like(q, 20.0), 2 * A * a2 / w2 + 1
    off = torch.where(2 * q < 0.1249, series, torch.where(2 * q > 0.1251, difference, torch.maximum(series, difference)))
    W = off / 2 + 2
    want = w * si * X
    assert ((out.double() - want).abs() <= (W + 15) * N * want.abs()).all()
    for t in range(min(T, 3)):
        _, step = gated_scan_step(*(v.detach()[:, t] for v in leaves), rate, torch.randn(B, F, device="cuda"), done[:, t])
        assert ((step.double() - want[:, t]).abs() <= (W + 15)[:, t] * N * want[:, t].abs()).all()
    for got, exp, tol in ((dx, G * w * si, W + 16), (di, G * want * (1 - si), W + 33),
                          (dd, G * a2 * si * X / w * q * (1 - sd), W + 2 * A + 49)):
        assert ((got.double() - exp).abs() <= tol * N * exp.abs() + 1e-37).all()

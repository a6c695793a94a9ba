"""Pins the oracle of the gated recurrence (oracle/gated.py) by finite differences and special cases."""
import numpy as np

from oracle import gated as og


def problem(seed, B=2, T=5, F=3):
    rng = np.random.default_rng(seed)
    x, i, d, dout = rng.standard_normal((4, B, T, F))
    rate = np.exp(rng.uniform(-3, 1, F))
    carry, dfinal = rng.standard_normal((2, B, F))
    return dict(x=x, input_gate=i, decay_gate=d, rate=rate, carry=carry), dfinal, dout


def test_vjp_matches_finite_differences():
    args, dfinal, dout = problem(1)
    done = np.zeros((2, 5), bool)
    done[0, 2] = done[1, 0] = done[1, 4] = True
    lengths = np.array([5, 3])

    def f(a):
        final, out, _ = og.gated_scan(*a.values(), done, lengths)
        return float((dfinal * final).sum() + (dout * out).sum())

    grads = og.gated_scan_vjp(*args.values(), done, lengths, dfinal, dout)
    for name, v in args.items():
        num = np.zeros_like(v)
        for i in np.ndindex(v.shape):
            moved = {n: u.copy() for n, u in args.items()}
            moved[name][i] += 1e-6
            up = f(moved)
            moved[name][i] -= 2e-6
            num[i] = (up - f(moved)) / 2e-6
        np.testing.assert_allclose(grads[name], num, rtol=1e-6, atol=1e-8)


def test_special_cases():
    args, _, _ = problem(2)
    shut = dict(args, input_gate=np.full((2, 5, 3), -800.0), decay_gate=np.full((2, 5, 3), 800.0))
    final, out, _ = og.gated_scan(*shut.values())
    np.testing.assert_allclose(final, np.exp(-5 * args["rate"]) * args["carry"], rtol=1e-12)   # no input: decay alone
    done = np.ones((2, 5), bool)
    g = og.gates(*(args[n] for n in ("x", "input_gate", "decay_gate", "rate")))
    _, out, before = og.gated_scan(*args.values(), done)
    np.testing.assert_array_equal(out, g["w"] * g["i"] * args["x"])                             # nothing is kept
    assert not before.any()
    final, out, _ = og.gated_scan(*args.values(), None, np.array([0, 5]))
    np.testing.assert_array_equal(final[0], args["carry"][0])
    assert not out[0].any()
    # unit inputs keep a unit variance: a^2 + w^2 = 1
    np.testing.assert_allclose(g["a"] ** 2 + g["w"] ** 2, 1, rtol=1e-12)

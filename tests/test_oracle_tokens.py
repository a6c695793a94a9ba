"""Pins the oracle of token log probabilities (oracle/tokens.py) by finite differences and special cases."""
import numpy as np

from oracle import tokens as otok


def test_vjp_matches_finite_differences():
    rng = np.random.default_rng(0)
    x = 2 * rng.standard_normal((2, 3, 5))
    mask = rng.random((2, 3, 5)) < 0.7
    mask[0, 0], mask[0, 1] = True, False
    tokens = np.array([[1, 2, -1], [4, 0, 9]])
    mask[1, 0, 4], mask[1, 1, 0] = True, False    # a token that is not allowed
    g, h = rng.standard_normal((2, 2, 3))

    def f(v):
        lp, H = otok.log_probs(v, tokens, mask, 0.7)
        return float((g * np.where(lp > -np.inf, lp, 0)).sum() + (h * H).sum())

    want, num = otok.vjp(x, tokens, g, h, mask, 0.7), np.zeros_like(x)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += 1e-6
        down[i] -= 1e-6
        num[i] = (f(up) - f(down)) / 2e-6
    np.testing.assert_allclose(want, num, rtol=1e-6, atol=1e-8)
    assert not want[~mask].any()


def test_special_rows():
    x = np.zeros((2, 1, 4))
    lp, H = otok.log_probs(x, np.array([[3], [7]]), None)
    np.testing.assert_allclose(lp, [[-np.log(4)], [0]])
    np.testing.assert_allclose(H, np.log(4))
    mask = np.array([[[False] * 4], [[True, False, True, False]]])
    lp, H = otok.log_probs(x, np.array([[0], [1]]), mask)
    assert (lp == -np.inf).all()
    np.testing.assert_allclose(H[:, 0], [0, np.log(2)])
    best, which = otok.top(x, 3, mask)
    np.testing.assert_array_equal(which[:, 0], [[-1, -1, -1], [0, 2, -1]])
    np.testing.assert_allclose(best[1, 0], [-np.log(2), -np.log(2), -np.inf])

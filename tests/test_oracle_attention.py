"""The float64 oracle of linear attention and of the query / key norms with
rotation: its gradients against central differences, and the chunk identity
that the kernels use against the recurrence."""
import numpy as np
import pytest

from oracle import attention as oat


def _difference(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        y = x.copy()
        y[i] += h
        up = f(y)
        y[i] -= 2 * h
        g[i] = (up - f(y)) / (2 * h)
    return g


@pytest.mark.parametrize("lengths", [None, [5, 0, 3]])
def test_linear_attention_gradients_match_differences(lengths):
    rng = np.random.default_rng(0)
    B, T, H, G, K, V = 3, 5, 4, 2, 2, 3
    q, k, v = rng.normal(size=(B, T, H, K)), rng.normal(size=(B, T, G, K)), rng.normal(size=(B, T, G, V))
    carry, g = rng.normal(size=(B, H, K, V)), -rng.random(H)
    done = rng.random((B, T)) < 0.3
    dfinal, dout = rng.normal(size=(B, H, K, V)), rng.normal(size=(B, T, H, V))

    def loss(q, k, v, carry):
        final, out = oat.linear_attention(q, k, v, g, carry, done, lengths, 0.7)
        return (final * dfinal).sum() + (out * dout).sum()

    got = oat.linear_attention_vjp(q, k, v, g, carry, done, lengths, 0.7, dfinal, dout)
    args = [q, k, v, carry]
    for n in range(4):
        want = _difference(lambda x: loss(*[x if i == n else a for i, a in enumerate(args)]), args[n])
        np.testing.assert_allclose(got[n], want, atol=1e-8)


def test_a_chunk_is_its_pair_sums_and_its_entry_state():
    rng = np.random.default_rng(1)
    T, K, V, g = 9, 3, 4, -0.2
    q, k, v = rng.normal(size=(1, T, 1, K)), rng.normal(size=(1, T, 1, K)), rng.normal(size=(1, T, 1, V))
    carry = rng.normal(size=(1, 1, K, V))
    done = np.zeros((1, T), bool)
    done[0, 4] = True
    final, out = oat.linear_attention(q, k, v, [g], carry, done)
    i = np.arange(T)
    start = np.where(i >= 4, 4, 0)
    w = np.where((i[:, None] >= i) & (i >= start[:, None]), np.exp(g * (i[:, None] - i)), 0)
    entry = np.where(i < 4, np.exp(g * (i + 1)), 0)[:, None]
    pairs = (w * (q[0, :, 0] @ k[0, :, 0].T)) @ v[0, :, 0]
    np.testing.assert_allclose(out[0, :, 0], pairs + entry * (q[0, :, 0] @ carry[0, 0]), atol=1e-12)
    tail = np.where(i >= 4, np.exp(g * (T - 1 - i)), 0)[:, None]
    np.testing.assert_allclose(final[0, 0], (tail * k[0, :, 0]).T @ v[0, :, 0], atol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_gradients_match_differences(interleaved):
    rng = np.random.default_rng(2)
    x, scale, cot = rng.normal(size=(2, 3, 2, 7)), rng.normal(size=7), rng.normal(size=(2, 3, 2, 7))
    f, pos = np.array([1.0, 0.1, 0.02]), rng.integers(0, 1000, (2, 3))
    dx, dscale = oat.norm_rotary_vjp(x, scale, f, pos, 1e-6, interleaved, cot)
    np.testing.assert_allclose(
        dx, _difference(lambda y: (oat.norm_rotary(y, scale, f, pos, 1e-6, interleaved) * cot).sum(), x), atol=1e-8)
    np.testing.assert_allclose(
        dscale, _difference(lambda y: (oat.norm_rotary(x, y, f, pos, 1e-6, interleaved) * cot).sum(), scale), atol=1e-8)


def _bf16(x):
    bits = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((bits + 0x7fff + (bits >> 16 & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).astype(np.float64)


def _pieces(x, count):
    """The sum of the bf16 values nearest to x and to what the ones before leave."""
    x, total = np.asarray(x, np.float32).astype(np.float64), 0.0
    for _ in range(count):
        p = _bf16(x)
        x, total = x - p, total + p
    return total


@pytest.mark.parametrize("width", [32, 128])
def test_the_norms_bounds_tell_one_piece_from_two_and_two_from_three(width):
    """What the bounds of test_gpu_attention_precision.py see: a state whose
    decayed terms keep two bf16 pieces is outside the float32 bound, with three
    inside; outputs whose pair products keep one piece before bf16's own
    rounding are outside the bf16 bounds, with two inside."""
    rng = np.random.default_rng(2)
    T, g = 300, -0.003
    q, k, v = (_bf16(rng.normal(size=(T, width))) for _ in range(3))
    i = np.arange(T)
    w = np.exp(g * (T - 1 - i)).astype(np.float32).astype(np.float64)
    state = k.T @ (v * w[:, None])
    off = [np.linalg.norm(k.T @ _pieces(v * w[:, None], n) - state) / np.linalg.norm(state) for n in (2, 3)]
    assert off[1] < 1e-7 and 1e-6 < off[0] < 1e-5
    weights = np.where(i[:, None] >= i, np.exp(g * (i[:, None] - i)), 0) * width ** -0.5
    pairs, terms = (q @ k.T) * weights, (np.abs(q) @ np.abs(k.T) * weights) @ np.abs(v)
    out = pairs @ v
    for n, inside in ((1, False), (2, True)):
        off = np.abs(_bf16(_pieces(pairs, n) @ v) - out)
        tol = 2.0 ** -16 * terms
        assert (off <= tol + 2.0 ** -8 * (np.abs(out) + tol)).all() == inside
        assert (np.linalg.norm(off) <= 2.0 ** -8 / 3 ** 0.5 * np.linalg.norm(out)) == inside

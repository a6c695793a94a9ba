"""Pins the oracle of the norms around a block (oracle/residual.py) by finite differences and special cases."""
import numpy as np
import pytest

from oracle import residual as ores


def problem(seed, D=7):
    rng = np.random.default_rng(seed)
    u, x, g, dy, dz = rng.standard_normal((5, 2, 3, D))
    post, scale, pre = 1 + 0.3 * rng.standard_normal((3, D))
    return dict(u=u, x=x, g=g, post=post, scale=scale, pre=pre), dy, dz


@pytest.mark.parametrize("post_norm", [True, False])
@pytest.mark.parametrize("gate", [None, "plain", "sigmoid"])
def test_vjp_matches_finite_differences(gate, post_norm):
    args, dy, dz = problem(1)
    if gate is None:
        args["g"] = None
    tail = (post_norm, gate == "sigmoid", 1e-3)

    def f(a):
        y, z = ores.residual_norm(*a.values(), *tail)
        return float((dy * y).sum() + (dz * z).sum())

    grads = ores.residual_norm_vjp(*args.values(), *tail, dy, dz)
    for name, key in (("u", "block"), ("x", "residual"), ("g", "gate"), ("post", "post"), ("scale", "scale"), ("pre", "pre")):
        if args[name] is None:
            continue
        num = np.zeros_like(args[name])
        for i in np.ndindex(num.shape):
            moved = {n: None if v is None else v.copy() for n, v in args.items()}
            moved[name][i] += 1e-6
            up = f(moved)
            moved[name][i] -= 2e-6
            num[i] = (up - f(moved)) / 2e-6
        np.testing.assert_allclose(grads[key], num, rtol=1e-6, atol=1e-7)


def test_a_stream_without_its_block_is_normed_alone():
    args, _, _ = problem(2)
    y, z = ores.residual_norm(*dict(args, scale=np.zeros(7)).values(), True, True, 1e-6)
    np.testing.assert_array_equal(y, args["x"])
    np.testing.assert_allclose((z / args["pre"]) ** 2 @ np.ones(7) / 7, 1, rtol=1e-5)

"""Oracle of the norms around a block — TEST INFRASTRUCTURE ONLY.

float64 numpy, rows along the last axis: n = u / rms(u) post (or u), y = x +
scale gate n, z = y / rms(y) pre, with rms(v) = sqrt(mean(v^2) + epsilon), and
the gradients of sum(dy y) + sum(dz z).  Pinned by finite differences
(tests/test_oracle_residual.py)."""
from __future__ import annotations

import numpy as np


def _rstd(v, epsilon):
    return 1 / np.sqrt((v * v).mean(-1, keepdims=True) + epsilon)


def parts(u, x, g, post, scale, pre, post_norm, sigmoid, epsilon):
    """What both directions need, by name."""
    gate = np.ones_like(u) if g is None else 1 / (1 + np.exp(-g)) if sigmoid else g
    ru = _rstd(u, epsilon) if post_norm else np.ones_like(u[..., :1])
    un = u * ru
    n = un * post
    y = x + scale * gate * n
    ry = _rstd(y, epsilon)
    return dict(gate=gate, ru=ru, un=un, n=n, y=y, ry=ry, yn=y * ry)


def residual_norm(u, x, g, post, scale, pre, post_norm, sigmoid, epsilon):
    p = parts(u, x, g, post, scale, pre, post_norm, sigmoid, epsilon)
    return p["y"], p["yn"] * pre


def residual_norm_vjp(u, x, g, post, scale, pre, post_norm, sigmoid, epsilon, dy, dz):
    """By name: block, residual, gate, post, scale, pre."""
    p = parts(u, x, g, post, scale, pre, post_norm, sigmoid, epsilon)
    rows = tuple(range(u.ndim - 1))
    e = dz * pre
    dx = dy + p["ry"] * (e - p["yn"] * (e * p["yn"]).mean(-1, keepdims=True))
    slope = p["gate"] * (1 - p["gate"]) if sigmoid else 1.0
    dn = dx * scale * p["gate"]
    f = dn * post
    du = p["ru"] * (f - p["un"] * (f * p["un"]).mean(-1, keepdims=True)) if post_norm else f
    return dict(block=du, residual=dx, gate=dx * scale * p["n"] * slope, post=(dn * p["un"]).sum(rows),
                scale=(dx * p["gate"] * p["n"]).sum(rows), pre=(dz * p["yn"]).sum(rows))

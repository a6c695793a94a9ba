"""Oracle of the gated linear recurrence — TEST INFRASTRUCTURE ONLY.

float64 numpy, step after step: a = exp(-rate sigmoid(decay_gate)), w = sqrt(1 -
a^2), h_t = a_t (done_t ? 0 : h_{t-1}) + w_t sigmoid(input_gate_t) x_t for t <
lengths, and the gradients of sum(dout h) + sum(dfinal final).  Pinned by finite
differences (tests/test_oracle_gated.py)."""
from __future__ import annotations

import numpy as np


def gates(x, input_gate, decay_gate, rate):
    """By name: i, r, a, w, and q = rate r."""
    i, r = 1 / (1 + np.exp(-input_gate)), 1 / (1 + np.exp(-decay_gate))
    q = rate * r
    return dict(i=i, r=r, q=q, a=np.exp(-q), w=np.sqrt(-np.expm1(-2 * q)))


def _kept(x, done, lengths):
    """Masks [batch, steps, 1]: steps inside a sequence, and those that keep the state before them."""
    B, T = x.shape[:2]
    inside = np.ones((B, T), bool) if lengths is None else np.arange(T) < np.asarray(lengths)[:, None]
    kept = inside if done is None else inside & ~np.asarray(done, bool)
    return inside[..., None], kept[..., None]


def gated_scan(x, input_gate, decay_gate, rate, carry=None, done=None, lengths=None):
    """(final, outputs, states before each step: 0 where the step starts an episode)"""
    g = gates(x, input_gate, decay_gate, rate)
    inside, kept = _kept(x, done, lengths)
    h = np.zeros((x.shape[0], x.shape[2])) if carry is None else np.array(carry, np.float64)
    out, before = np.zeros_like(x), np.zeros_like(x)
    for t in range(x.shape[1]):
        before[:, t] = np.where(kept[:, t], h, 0)
        new = g["a"][:, t] * before[:, t] + (g["w"] * g["i"] * x)[:, t]
        h = np.where(inside[:, t], new, h)
        out[:, t] = np.where(inside[:, t], new, 0)
    return h, out, before


def gated_scan_vjp(x, input_gate, decay_gate, rate, carry, done, lengths, dfinal, dout):
    """By name: x, input_gate, decay_gate, rate, carry; and D, the cotangent of each step's state."""
    g = gates(x, input_gate, decay_gate, rate)
    inside, kept = _kept(x, done, lengths)
    _, _, before = gated_scan(x, input_gate, decay_gate, rate, carry, done, lengths)
    E, D = np.array(dfinal, np.float64), np.zeros_like(x)
    for t in range(x.shape[1] - 1, -1, -1):
        d = dout[:, t] + E
        D[:, t] = np.where(inside[:, t], d, 0)
        E = np.where(inside[:, t], np.where(kept[:, t], g["a"][:, t] * d, 0), E)
    i, r, a, w = (g[n] for n in "iraw")
    dL = D * (a * before - a * a * i * x / w)
    return dict(x=D * w * i, input_gate=D * w * x * i * (1 - i), decay_gate=dL * -rate * r * (1 - r),
                rate=(-dL * r).sum((0, 1)), carry=E, D=D)

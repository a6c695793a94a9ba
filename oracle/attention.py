"""Linear attention with a decay for each head and the query / key norms with
rotation, in numpy float64, step by step from their definitions, with their
vector-Jacobian products written out."""
from __future__ import annotations

import numpy as np


def _prepare(q, k, v, log_decay, carry, done, lengths):
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, T, H, K = q.shape
    V = v.shape[-1]
    of = np.arange(H) // (H // k.shape[2])
    lam = np.exp(np.asarray(log_decay, np.float64))
    carry = np.zeros((B, H, K, V)) if carry is None else np.asarray(carry, np.float64)
    done = np.zeros((B, T), bool) if done is None else np.asarray(done)
    lengths = np.full(B, T) if lengths is None else np.clip(np.asarray(lengths), 0, T)
    return q, k, v, of, lam, carry, done, lengths


def linear_attention(q, k, v, log_decay, carry=None, done=None, lengths=None, scale=1.0, states=None):
    """(final [B, H, K, V], out [B, T, H, V]); every state into the list `states` where given."""
    q, k, v, of, lam, carry, done, lengths = _prepare(q, k, v, log_decay, carry, done, lengths)
    B, T, H, _ = q.shape
    out = np.zeros((B, T, H, v.shape[-1]))
    final = carry.copy()
    for b in range(B):
        S = carry[b]
        for t in range(lengths[b]):
            before = np.zeros_like(S) if done[b, t] else lam[:, None, None] * S
            S = before + k[b, t, of][:, :, None] * v[b, t, of][:, None, :]
            out[b, t] = scale * (q[b, t][:, None, :] @ S)[:, 0]
            if states is not None:
                states.append(S)
        final[b] = S
    return final, out


def linear_attention_vjp(q, k, v, log_decay, carry, done, lengths, scale, dfinal, dout):
    """(dq, dk, dv, dcarry)."""
    states = []
    linear_attention(q, k, v, log_decay, carry, done, lengths, scale, states)
    q, k, v, of, lam, carry, done, lengths = _prepare(q, k, v, log_decay, carry, done, lengths)
    dout = np.asarray(dout, np.float64)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    dcarry = np.zeros_like(carry) if dfinal is None else np.array(dfinal, np.float64)
    at = 0
    for b in range(q.shape[0]):
        D = dcarry[b]
        for t in reversed(range(lengths[b])):
            S = states[at + t]
            D = D + scale * q[b, t][:, :, None] * dout[b, t][:, None, :]
            dq[b, t] = scale * (S @ dout[b, t][:, :, None])[..., 0]
            np.add.at(dk[b, t], of, (D @ v[b, t, of][:, :, None])[..., 0])
            np.add.at(dv[b, t], of, (k[b, t, of][:, None, :] @ D)[:, 0])
            D = np.zeros_like(D) if done[b, t] else lam[:, None, None] * D
        dcarry[b] = D
        at += lengths[b]
    return dq, dk, dv, dcarry


def _columns(pairs, interleaved):
    i = np.arange(pairs)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)


def _turn(x, frequencies, positions, interleaved, sign):
    first, second = _columns(len(frequencies), interleaved)
    angle = np.asarray(positions, np.float64)[..., None, None] * np.asarray(frequencies, np.float64)
    c, s = np.cos(angle), sign * np.sin(angle)
    out = x.copy()
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., second] * c + x[..., first] * s
    return out


def norm_rotary(x, scale, frequencies, positions, epsilon, interleaved=False):
    """x [B, T, heads, D], scale [D], positions [B, T]."""
    x = np.asarray(x, np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)
    return _turn(x * r * np.asarray(scale, np.float64), frequencies, positions, interleaved, 1.0)


def norm_rotary_vjp(x, scale, frequencies, positions, epsilon, interleaved, cot):
    """(dx, dscale)."""
    x, scale = np.asarray(x, np.float64), np.asarray(scale, np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)
    e = _turn(np.asarray(cot, np.float64), frequencies, positions, interleaved, -1.0)
    dscale = (e * x * r).reshape(-1, x.shape[-1]).sum(0)
    e = e * scale
    return r * (e - x * r * r * (e * x).mean(-1, keepdims=True)), dscale

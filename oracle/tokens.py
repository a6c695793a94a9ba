"""Oracle of token log probabilities — TEST INFRASTRUCTURE ONLY.

float64 numpy: of softmax(logits / temperature) with -inf where the mask does
not allow, the log probability of a token (none: 0; not allowed: -inf), the
entropy, the best alternatives in falling order (equal ones by index, -1 and
-inf past the allowed), and the gradient of sum(g log_prob) + sum(h entropy),
to which tokens that are none or not allowed add nothing.  Pinned by finite
differences (tests/test_oracle_tokens.py)."""
from __future__ import annotations

import numpy as np


def masked(logits, mask):
    x = np.asarray(logits, np.float64)
    return x if mask is None else np.where(mask, x, -np.inf)


def log_softmax(x, temperature):
    """log p and the rows that allow something (others: -inf everywhere)."""
    m = x.max(-1, keepdims=True)
    some = m > -np.inf
    with np.errstate(invalid="ignore", divide="ignore"):
        w = (x - np.where(some, m, 0)) / temperature
        return np.where(some, w - np.log(np.exp(w).sum(-1, keepdims=True)), -np.inf), some[..., 0]


def _given(tokens, vocab):
    inside = (tokens >= 0) & (tokens < vocab)
    return inside, np.where(inside, tokens, 0)[..., None]


def log_probs(logits, tokens, mask=None, temperature=1.0):
    """(log_prob, entropy)"""
    logp, _ = log_softmax(masked(logits, mask), temperature)
    inside, at = _given(tokens, logp.shape[-1])
    p = np.exp(logp)
    entropy = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(-1)
    return np.where(inside, np.take_along_axis(logp, at, -1)[..., 0], 0.0), entropy


def top(logits, count, mask=None, temperature=1.0):
    """(log probabilities, tokens)"""
    x = masked(logits, mask)
    logp, _ = log_softmax(x, temperature)
    order = np.argsort(-x, axis=-1, kind="stable")[..., :count]
    best = np.take_along_axis(logp, order, -1)
    none = np.take_along_axis(x, order, -1) == -np.inf
    return np.where(none, -np.inf, best), np.where(none, -1, order)


def vjp(logits, tokens, g, h, mask=None, temperature=1.0):
    logp, _ = log_softmax(masked(logits, mask), temperature)
    log_prob, entropy = log_probs(logits, tokens, mask, temperature)
    inside, at = _given(tokens, logp.shape[-1])
    g = np.where(inside & (log_prob > -np.inf), g, 0.0)[..., None]
    p = np.exp(logp)
    d = -p * (g + h[..., None] * np.where(p > 0, logp + entropy[..., None], 0))
    np.put_along_axis(d, at, np.take_along_axis(d, at, -1) + g, -1)
    return d / temperature

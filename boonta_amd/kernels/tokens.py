"""Log probabilities of given tokens with the entropy and the top alternatives
on MI355X: what a policy over tokens, or over any number of discrete actions,
takes from its logits (boonta/networks/distributions.py:8-38, whose categorical
the learners' fused heads compute for a few dozen actions).

- ``token_log_probs(logits, tokens, mask, temperature, top)`` ->
  ``TokenLogProbs(log_prob, entropy, top_log_probs, top_tokens)``; log_prob and
  entropy are differentiable in the logits.

float32 or bfloat16 logits; sums and results are float32, and gradients are
rounded to the logits' type once.  There is no CPU path.  It runs on the device
the tensors live on, on its current stream, and can be captured into a graph
(drop every eager autograd graph of the same leaves first, as for
``linear_attention``).  Forward-mode tangents are refused.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .attention import _DTYPES, _launch, _no_tangents, _on_device, _ptr, _rows

_TOKENS = {torch.int32: 0, torch.int64: 1}


class TokenLogProbs(NamedTuple):
    log_prob: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor | None = None
    top_tokens: torch.Tensor | None = None


_STRIDES = {n: ctypes.c_int64 * n for n in (4, 8)}


def _strides(dims, *tensors):
    flat = []
    for x in tensors:
        s = (0, 0) if x is None else x.stride()[:dims]
        flat += s if dims == 2 else (s[0], 0)
    return _STRIDES[len(flat)](*flat)


def _forward(logits, tokens, mask, temperature, top, keep):
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    batch, steps = lead if len(lead) == 2 else (lead[0], 1)
    log_prob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(log_prob)
    stats = log_prob.new_empty((*lead, 2)) if keep else None
    top_log_probs = log_prob.new_empty((*lead, top)) if top else None
    top_tokens = tokens.new_empty((*lead, top)) if top else None
    nbytes = _lib.load().ppo_token_log_probs_workspace(batch, steps, vocab, top)
    work = log_prob.new_empty(nbytes // 4) if nbytes else None
    _launch(logits.get_device(), "ppo_token_log_probs_fwd", _DTYPES[logits.dtype], logits.data_ptr(),
            tokens.data_ptr(), _TOKENS[tokens.dtype], _ptr(mask), _strides(len(lead), logits, mask), temperature, top,
            log_prob.data_ptr(), entropy.data_ptr(), _ptr(stats), _ptr(top_log_probs), _ptr(top_tokens), _ptr(work),
            nbytes, batch, steps, vocab)
    return log_prob, entropy, top_log_probs, top_tokens, stats


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, top):
        *outs, stats = _forward(logits, tokens, mask, temperature, top, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(x for x in outs[2:] if x is not None))
        ctx.save_for_backward(logits, tokens, mask, outs[0], outs[1], stats)
        ctx.temperature = temperature
        return tuple(outs)

    @staticmethod
    @once_differentiable
    def backward(ctx, dlog_prob, dentropy, *_):
        _no_tangents("token_log_probs", dlog_prob, dentropy)
        logits, tokens, mask, log_prob, entropy, stats = ctx.saved_tensors
        lead, vocab = logits.shape[:-1], logits.shape[-1]
        batch, steps = lead if len(lead) == 2 else (lead[0], 1)
        dlogits = logits.new_empty(logits.shape)
        _launch(logits.get_device(), "ppo_token_log_probs_bwd", _DTYPES[logits.dtype], logits.data_ptr(),
                tokens.data_ptr(), _TOKENS[tokens.dtype], _ptr(mask),
                _strides(len(lead), logits, mask, dlog_prob, dentropy), ctx.temperature, log_prob.data_ptr(),
                entropy.data_ptr(), stats.data_ptr(), _ptr(dlog_prob), _ptr(dentropy), dlogits.data_ptr(), batch, steps,
                vocab)
        return dlogits, None, None, None, None


_limits = None


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, mask: torch.Tensor | None = None,
                    temperature: float = 1.0, top: int = 0) -> TokenLogProbs:
    """Of the categorical distributions softmax(logits / temperature) over the last axis:

    - log_prob: of ``tokens``, -inf where the token is not allowed (or where the
      value of an allowed one is below float32's range: its gradient is that of
      any other); a token outside the vocabulary (-1, say) is none: its log_prob
      is 0 and passes no gradient;
    - entropy (0 where nothing is allowed);
    - top_log_probs, top_tokens: the ``top`` most probable tokens in falling
      order, equal ones by index, without gradients; past the allowed ones -inf
      and -1.  None without ``top``.

    logits [batch, steps, vocab] or [batch, vocab] in any strides, float32 or
    bfloat16; tokens int32 or int64 of the leading shape; mask: bool, broadcast to
    the logits, False (as a logit of -inf) where a token is not allowed: what is
    there, NaN among it, counts nowhere, and gets no gradient, whatever the
    cotangents.  A token that is not allowed passes no gradient.  +inf or NaN
    among the allowed makes its row's results NaN.  Results are float32 of the leading shape, top_tokens
    of the tokens' type.  Vocabularies up to 2^24, ``top`` up to 32 and the vocabulary,
    2^24 - 1 rows."""
    global _limits
    if _limits is None:
        lib = _lib.load()
        _limits = lib.ppo_token_log_probs_max_top(), lib.ppo_token_log_probs_max_vocab()
    shape = logits.shape
    if logits.dtype not in _DTYPES:
        raise TypeError(f"token_log_probs takes float32 or bfloat16 logits, not {logits.dtype}")
    if tokens.dtype not in _TOKENS:
        raise TypeError(f"tokens must be int32 or int64, not {tokens.dtype}")
    if len(shape) not in (2, 3) or tokens.shape != shape[:-1]:
        raise ValueError(f"need logits [batch, steps, vocab] or [batch, vocab] and tokens of their leading shape; got "
                         f"{tuple(shape)}, {tuple(tokens.shape)}")
    if not 0 < shape[-1] <= _limits[1]:
        raise ValueError(f"token_log_probs takes vocabularies from 1 up to {_limits[1]}, not {shape[-1]}")
    temperature, top = float(temperature), int(top)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be above 0 (from 1e-30 to 1e30), not {temperature}")
    if not 0 <= top <= min(_limits[0], shape[-1]):
        raise ValueError(f"top must be from 0 up to {min(_limits[0], shape[-1])}, not {top}")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"mask must be bool, not {mask.dtype}")
        if mask.shape != shape:
            try:
                mask = mask.expand(shape)
            except RuntimeError:
                raise ValueError(f"mask must broadcast to {tuple(shape)}, got {tuple(mask.shape)}") from None
    _on_device("token_log_probs", logits, tokens, mask)
    logits, tokens = _rows(logits), tokens.contiguous()
    mask = None if mask is None else _rows(mask)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, mask, temperature, top))
    return TokenLogProbs(*_forward(logits, tokens, mask, temperature, top, False)[:4])

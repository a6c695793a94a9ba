"""The norms around a block of a residual torso on MI355X, with the block's gate,
the residual scale and the sum into the stream in the same pass.  It has no
counterpart in the reference, whose blocks are norms, gates and sums apart
(boonta/networks/blocks).

- ``residual_norm(block, residual, gate, post_scale, residual_scale, pre_scale)``
  -> (stream, normed): the new residual stream and its norm, which the next
  block reads; differentiable in all six.

float32 or bfloat16 storage, the stream float32 or the block's; sums and norms
are float32, and outputs are rounded to their type once.  There is no CPU path.
It runs on the device the tensors live on, on its current stream, and can be
captured into a graph (drop every eager autograd graph of the same leaves first,
as for ``linear_attention``).  Forward-mode tangents are refused.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .attention import _DTYPES, _launch, _no_tangents, _on_device, _ptr, _rows

_max_width = 0


_STRIDES = {n: ctypes.c_int64 * n for n in (6, 10)}


def _strides(*tensors):
    flat = [s for x in tensors for s in ((0, 0) if x is None else x.stride()[:2])]
    return _STRIDES[len(flat)](*flat)


def _forward(block, residual, gate, post_scale, residual_scale, pre_scale, options, keep):
    post_norm, sigmoid, epsilon = options
    batch, steps, width = block.shape
    stream, normed = residual.new_empty(block.shape), block.new_empty(block.shape)
    stats = torch.empty((batch, steps, 2), dtype=torch.float32, device=block.device) if keep else None
    _launch(block.get_device(), "ppo_residual_norm_fwd", _DTYPES[block.dtype], _DTYPES[residual.dtype],
            block.data_ptr(), residual.data_ptr(), _ptr(gate), _strides(block, residual, gate), _ptr(post_scale),
            _ptr(residual_scale), _ptr(pre_scale), post_norm, sigmoid, epsilon, stream.data_ptr(), normed.data_ptr(),
            _ptr(stats), batch, steps, width)
    return stream, normed, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block, residual, gate, post_scale, residual_scale, pre_scale, options):
        stream, normed, stats = _forward(block, residual, gate, post_scale, residual_scale, pre_scale, options, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(block, residual, gate, post_scale, residual_scale, pre_scale, stats)
        ctx.options = options
        return stream, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, dstream, dnormed):
        _no_tangents("residual_norm", dstream, dnormed)
        block, residual, gate, *scales, stats = ctx.saved_tensors
        post_norm, sigmoid, _ = ctx.options
        batch, steps, width = block.shape
        dstream, dnormed = (None if x is None else _rows(x) for x in (dstream, dnormed))
        dblock, dresidual = block.new_empty(block.shape), residual.new_empty(block.shape)
        dgate = None if gate is None or not ctx.needs_input_grad[2] else gate.new_empty(block.shape)
        dscales = [None if x is None or not need else torch.empty_like(x)
                   for x, need in zip(scales, ctx.needs_input_grad[3:6])]
        nbytes, work = 0, None
        if any(x is not None for x in dscales):
            nbytes = _lib.load().ppo_residual_norm_bwd_workspace(_DTYPES[block.dtype], batch, steps, width)
            work = torch.empty(nbytes // 4, dtype=torch.float32, device=block.device)
        _launch(block.get_device(), "ppo_residual_norm_bwd", _DTYPES[block.dtype], _DTYPES[residual.dtype],
                block.data_ptr(), residual.data_ptr(), _ptr(gate), _ptr(dstream), _ptr(dnormed),
                _strides(block, residual, gate, dstream, dnormed), *map(_ptr, scales), post_norm, sigmoid,
                stats.data_ptr(), dblock.data_ptr(), dresidual.data_ptr(), _ptr(dgate), *map(_ptr, dscales),
                _ptr(work), nbytes, batch, steps, width)
        return dblock, dresidual, dgate, *dscales, None


def residual_norm(block: torch.Tensor, residual: torch.Tensor, gate: torch.Tensor | None = None,
                  post_scale: torch.Tensor | None = None, residual_scale: torch.Tensor | None = None,
                  pre_scale: torch.Tensor | None = None, post_norm: bool = True,
                  gate_activation: str | None = None, epsilon: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(stream, normed), both [batch, steps, width], of a block's output and the
    residual stream it is added to:

        n = block / sqrt(mean(block ** 2) + epsilon) * post_scale
        stream = residual + residual_scale * gate * n
        normed = stream / sqrt(mean(stream ** 2) + epsilon) * pre_scale

    means over the width, ``normed`` from the sum before it is rounded.  block and
    gate [batch, steps, width] in any strides, float32 or bfloat16, and normed
    as they; residual and stream of their type or float32.  gate: None (1), as it
    is, or through gate_activation "sigmoid".  Scales: float32 [width], None:
    ones.  post_norm False: n = block (and no post_scale).  Gradients reach
    every operand.  Widths up to 8192, batch * steps up to 2^31 - 2^20 - 1."""
    global _max_width
    _max_width = _max_width or _lib.load().ppo_residual_norm_max_width()
    dtype, shape = block.dtype, block.shape
    if dtype not in _DTYPES:
        raise TypeError(f"residual_norm stores float32 or bfloat16, not {dtype}")
    if residual.dtype not in (dtype, torch.float32):
        raise TypeError(f"residual must be float32 or of the block's type, not {residual.dtype}")
    if gate is not None and gate.dtype != dtype:
        raise TypeError("block and gate must share one dtype")
    if len(shape) != 3 or residual.shape != shape or (gate is not None and gate.shape != shape):
        shapes = ", ".join(str(tuple(x.shape)) for x in (block, residual, gate) if x is not None)
        raise ValueError(f"need block, residual (and gate) of one shape [batch, steps, width]; got {shapes}")
    if shape[2] > _max_width:
        raise ValueError(f"residual_norm takes widths up to {_max_width}, not {shape[2]}")
    if gate_activation not in (None, "sigmoid"):
        raise ValueError(f"gate_activation is None or 'sigmoid', not {gate_activation!r}")
    if gate_activation is not None and gate is None:
        raise ValueError("gate_activation without a gate")
    if post_scale is not None and not post_norm:
        raise ValueError("post_scale without post_norm")
    for name, x in (("post_scale", post_scale), ("residual_scale", residual_scale), ("pre_scale", pre_scale)):
        if x is not None and (x.dtype != torch.float32 or x.shape != shape[2:]):
            raise ValueError(f"{name} must be float32 [{shape[2]}], got {x.dtype} {tuple(x.shape)}")
    _on_device("residual_norm", block, residual, gate, post_scale, residual_scale, pre_scale)
    block, residual = _rows(block), _rows(residual)
    gate = None if gate is None else _rows(gate)
    scales = [None if x is None else x.contiguous() for x in (post_scale, residual_scale, pre_scale)]
    options = (int(post_norm), int(gate_activation is not None), float(epsilon))
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (block, residual, gate, *scales)):
        return _ResidualNorm.apply(block, residual, gate, *scales, options)
    return _forward(block, residual, gate, *scales, options, False)[:2]

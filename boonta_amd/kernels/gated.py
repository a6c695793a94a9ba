"""A gated linear recurrence on MI355X: the recurrence of ``scan`` / ``ssm`` with
its decays and input weights formed from gates in the same pass, as the cells of
boonta/networks/blocks form them before the scan.  It has no counterpart in the
reference.

- ``gated_scan(x, input_gate, decay_gate, rate, carry, done, lengths)`` ->
  (final carry, outputs): whole sequences (training minibatches, prompts),
  differentiable in x, the gates, rate and carry;
- ``gated_scan_step(x, input_gate, decay_gate, rate, carry, done)`` ->
  (carry, output): one rollout step.

float32 or bfloat16 storage; states, gates and sums are float32, and outputs are
rounded to their type once.  There is no CPU path.  The kernels run on the device
the tensors live on, on its current stream, and can be captured into a graph
(drop every eager autograd graph of the same leaves first, as for
``linear_attention``).  Forward-mode tangents are refused.

Limits, past which a call is refused: 2^21 sequences, 2^30 steps, 2^20
features, 2^29 batch * features.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .attention import _DTYPES, _launch, _near_rows, _no_tangents, _on_device, _ptr, _rows


_STRIDES = {n: ctypes.c_int64 * n for n in (3, 6, 8)}


def _strides(*tensors):
    flat = [s for x in tensors for s in x.stride()[:-1]]
    return _STRIDES[len(flat)](*flat)


def _check(name, x, input_gate, decay_gate, rate, carry, done, dims):
    dtype, shape = x.dtype, x.shape
    if dtype not in _DTYPES:
        raise TypeError(f"{name} stores float32 or bfloat16, not {dtype}")
    if input_gate.dtype != dtype or decay_gate.dtype != dtype:
        raise TypeError("x and the gates must share one dtype")
    if len(shape) != dims or input_gate.shape != shape or decay_gate.shape != shape:
        raise ValueError(f"need x, input_gate and decay_gate of one shape [batch, {'steps, ' if dims == 3 else ''}"
                         f"features]; got {tuple(shape)}, {tuple(input_gate.shape)}, {tuple(decay_gate.shape)}")
    if rate.dtype != torch.float32 or rate.shape != shape[-1:]:
        raise ValueError(f"rate must be float32 [{shape[-1]}], got {rate.dtype} {tuple(rate.shape)}")
    state = (shape[0], shape[-1])
    if carry is not None and (carry.dtype != torch.float32 or carry.shape != state):
        raise ValueError(f"carry must be float32 {state}, got {carry.dtype} {tuple(carry.shape)}")
    if done is not None and (done.dtype != torch.bool or done.shape != shape[:-1]):
        raise ValueError(f"done must be bool {tuple(shape[:-1])}, got {done.dtype} {tuple(done.shape)}")
    return shape


def _forward(x, input_gate, decay_gate, rate, carry, done, lengths, keep):
    batch, steps, features = x.shape
    dt, lib = _DTYPES[x.dtype], _lib.load()
    out = x.new_empty(x.shape)
    if steps == 0:
        return (rate.new_zeros((batch, features)) if carry is None else carry.clone()), out, None
    final = rate.new_empty((batch, features))
    states = rate.new_empty(lib.ppo_gated_scan_states(dt, batch, steps, features) // 4) if keep else None
    nbytes = lib.ppo_gated_scan_workspace(dt, batch, steps, features)
    work = rate.new_empty(nbytes // 4) if nbytes else None
    _launch(x.get_device(), "ppo_gated_scan_fwd", dt, x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(),
            _strides(x, input_gate, decay_gate), rate.data_ptr(), _ptr(carry), _ptr(done), _ptr(lengths), out.data_ptr(),
            final.data_ptr(), _ptr(states), _ptr(work), nbytes, batch, steps, features)
    return final, out, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, input_gate, decay_gate, rate, carry, done, lengths):
        final, out, states = _forward(x, input_gate, decay_gate, rate, carry, done, lengths, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, input_gate, decay_gate, rate, done, lengths, states)
        return final, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dfinal, dout):
        _no_tangents("gated_scan", dfinal, dout)
        x, input_gate, decay_gate, rate, done, lengths, states = ctx.saved_tensors
        batch, steps, features = x.shape
        dt = _DTYPES[x.dtype]
        need_rate, need_carry = ctx.needs_input_grad[3:5]
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx, dinput_gate, ddecay_gate = (x.new_empty(x.shape) for _ in range(3))
        if x.numel() == 0:
            dcarry = rate.new_zeros((batch, features)) if dfinal is None else dfinal
            return (dx, dinput_gate, ddecay_gate, torch.zeros_like(rate) if need_rate else None,
                    dcarry if need_carry else None, None, None)
        if dout is None:   # (only the final carry was used)
            dout = x.new_zeros(features).expand(x.shape)
        dout = _near_rows(dout)
        drate = torch.empty_like(rate) if need_rate else None
        dcarry = rate.new_empty((batch, features)) if need_carry else None
        nbytes = _lib.load().ppo_gated_scan_bwd_workspace(dt, batch, steps, features)
        work = rate.new_empty(nbytes // 4)
        _launch(x.get_device(), "ppo_gated_scan_bwd", dt, x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(),
                dout.data_ptr(), _strides(x, input_gate, decay_gate, dout), rate.data_ptr(), _ptr(done), _ptr(lengths),
                states.data_ptr(), _ptr(dfinal), dx.data_ptr(), dinput_gate.data_ptr(), ddecay_gate.data_ptr(),
                _ptr(drate), _ptr(dcarry), work.data_ptr(), nbytes, batch, steps, features)
        return dx, dinput_gate, ddecay_gate, drate, dcarry, None, None


def gated_scan(x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor, rate: torch.Tensor,
               carry: torch.Tensor | None = None, done: torch.Tensor | None = None,
               lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(final carry [batch, features] float32, outputs [batch, steps, features]) of

        a_t = exp(-rate * sigmoid(decay_gate_t))
        h_t = a_t * (0 where done_t else h_{t-1}) + sqrt(1 - a_t ** 2) * sigmoid(input_gate_t) * x_t

    with h_{-1} = carry (None: zeros).  x and the gates [batch, steps, features] in
    any strides, float32 or bfloat16; rate: float32 [features], at least 0 (0
    keeps the state, and the gradient through its input weight, which has no
    bound there, is taken as 0).  done: bool [batch, steps], the step starts an
    episode: nothing from before it passes, an infinity or NaN neither.  lengths:
    int32 [batch], steps of each sequence: what follows counts nowhere, and its
    outputs and gradients are zeros.  What the recurrence gives an infinity may
    come out as NaN."""
    shape = _check("gated_scan", x, input_gate, decay_gate, rate, carry, done, 3)
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != shape[:1]):
        raise ValueError(f"lengths must be int32 [{shape[0]}], got {lengths.dtype} {tuple(lengths.shape)}")
    _on_device("gated_scan", x, input_gate, decay_gate, rate, carry, done, lengths)
    args = (_near_rows(x), _near_rows(input_gate), _near_rows(decay_gate), rate.contiguous(),
            *(None if t is None else t.contiguous() for t in (carry, done, lengths)))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:5]):
        return _GatedScan.apply(*args)
    return _forward(*args, False)[:2]


def gated_scan_step(x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor, rate: torch.Tensor,
                    carry: torch.Tensor, done: torch.Tensor | None = None,
                    out_carry: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(carry, output [batch, features]) of one step of ``gated_scan``: x and the
    gates [batch, features], done [batch].  The new carry is written to
    ``out_carry`` where given (``carry`` itself: in place; else apart from it).
    Without gradients: a step that needs them is a sequence of one."""
    batch, features = _check("gated_scan_step", x, input_gate, decay_gate, rate, carry, done, 2)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, input_gate, decay_gate, rate, carry)):
        raise ValueError("gated_scan_step has no gradients: use gated_scan on a sequence of one step")
    if out_carry is not None and (out_carry.dtype != torch.float32 or out_carry.shape != carry.shape
                                  or not out_carry.is_contiguous() or out_carry.requires_grad):
        raise ValueError(f"out_carry must be contiguous float32 {tuple(carry.shape)} that needs no gradient")
    if out_carry is not None and 0 < abs(out_carry.data_ptr() - carry.data_ptr()) < 4 * carry.numel():
        raise ValueError("out_carry must be carry itself or memory apart from it")
    index = _on_device("gated_scan_step", x, input_gate, decay_gate, rate, carry, done, out_carry)
    x, input_gate, decay_gate, rate, carry = _rows(x), _rows(input_gate), _rows(decay_gate), rate.contiguous(), carry.contiguous()
    done = None if done is None else done.contiguous()
    if out_carry is None:
        out_carry = carry.new_empty((batch, features))
    else:
        torch.autograd.graph.increment_version(out_carry)   # (written in place)
    out = x.new_empty((batch, features))
    _launch(index, "ppo_gated_scan_step", _DTYPES[x.dtype], x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(),
            _strides(x, input_gate, decay_gate), rate.data_ptr(), carry.data_ptr(), _ptr(done), out.data_ptr(),
            out_carry.data_ptr(), batch, features)
    return out_carry, out

"""Linear attention with a decay for each head on MI355X, and the per-head norms
of queries and keys with the position rotation that feed it.  The recurrence
of ``scan`` / ``ssm`` with a matrix for a state; it has no counterpart in the
reference, whose attention block is boonta/networks/blocks/self_attention.py.

- ``linear_attention(q, k, v, log_decay, carry, done, lengths, scale)`` ->
  (final carry, outputs): whole sequences (training minibatches, prompts),
  differentiable in q, k, v and carry;
- ``linear_attention_step(q, k, v, log_decay, carry, done, scale)`` ->
  (carry, output): one rollout step;
- ``qk_norm_rotary(q, k, q_scale, k_scale, frequencies, positions)`` -> (q, k),
  differentiable in q, k and the scales; ``rotary_frequencies`` makes its
  usual frequencies.

float32 or bfloat16 storage; states, sums and norms are float32.  There is no CPU path:
the kernels run on the device the tensors live on, on its current stream.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable
from torch.nn.functional import pad

from .. import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_MAX_STRIDE = 1 << 23   # of a step, in elements: the kernels count a chunk's bytes in 32 bits


def _on_device(name, *tensors):
    device = tensors[0].device
    for x in tensors:
        if x is not None and (not x.is_cuda or x.device != device):
            raise TypeError(f"{name} runs on tensors of one device")
    return device


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # (a build without devices has none)


def _launch(device, name, *args):
    """Calls an entry point on the device's current stream (the device made current where it is not)."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, _raw_stream(device.index), *args)
    else:
        with torch.cuda.device(device):
            _lib.call(name, _raw_stream(device.index), *args)


def _rows(x):
    """x, or a copy where its columns are not side by side or its rows too far apart."""
    st = x.stride()
    if (st[-1] != 1 and x.shape[-1] > 1) or (x.dim() == 4 and st[1] > _MAX_STRIDE):
        return x.contiguous()
    return x


def _strides(*tensors):
    flat = [s for x in tensors for s in x.stride()[:-1]]
    return (ctypes.c_int64 * len(flat))(*flat)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _check_heads(name, q, k, v, dims):
    if q.dtype not in _DTYPES:
        raise TypeError(f"{name} stores float32 or bfloat16, not {q.dtype}")
    if k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise TypeError("q, k and v must share one dtype" if v is not None else "q and k must share one dtype")
    lead = dims - 2
    ok = q.dim() == dims and k.dim() == dims and k.shape[:lead] == q.shape[:lead] and k.shape[-1] == q.shape[-1]
    if v is not None:
        ok = ok and v.dim() == dims and v.shape[:-1] == k.shape[:-1]
    if not ok:
        shapes = ", ".join(str(tuple(x.shape)) for x in (q, k, v) if x is not None)
        raise ValueError(f"need q [{'batch, steps' if dims == 4 else 'batch'}, heads, width], k (and v) of the same "
                         f"batch{' and steps' if dims == 4 else ''} with heads that divide q's; got {shapes}")


def _check_attention(name, q, k, v, log_decay, carry, done, dims):
    _check_heads(name, q, k, v, dims)
    heads, kv_heads = q.shape[-2], k.shape[-2]
    if (kv_heads == 0) != (heads == 0) or (heads and heads % kv_heads):
        raise ValueError(f"{heads} heads do not share {kv_heads} key heads evenly")
    limit = _lib.load().ppo_linear_attention_max_width()
    if not (0 < q.shape[-1] <= limit and 0 < v.shape[-1] <= limit):
        raise ValueError(f"{name} takes widths from 1 up to {limit}, not {q.shape[-1]} and {v.shape[-1]}")
    if log_decay.dtype != torch.float32 or tuple(log_decay.shape) != (heads,):
        raise ValueError(f"log_decay must be float32 [{heads}], got {log_decay.dtype} {tuple(log_decay.shape)}")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a fixed schedule: it gets no gradient, pass it detached")
    shape = (q.shape[0], heads, q.shape[-1], v.shape[-1])
    if carry is not None and (carry.dtype != torch.float32 or tuple(carry.shape) != shape):
        raise ValueError(f"carry must be float32 {shape}, got {carry.dtype} {tuple(carry.shape)}")
    if done is not None and (done.dtype != torch.bool or done.shape != q.shape[:dims - 2]):
        raise ValueError(f"done must be bool {tuple(q.shape[:dims - 2])}, got {done.dtype} {tuple(done.shape)}")


# --------------------------------------------------------------------- sequences
def _forward(q, k, v, log_decay, carry, done, lengths, scale):
    batch, steps, heads, key = q.shape
    kv_heads, value = v.shape[-2:]
    device, dt = q.device, _DTYPES[q.dtype]
    out = torch.empty((batch, steps, heads, value), dtype=q.dtype, device=device)
    final = torch.empty((batch, heads, key, value), dtype=torch.float32, device=device)
    nbytes = _lib.load().ppo_linear_attention_workspace(dt, batch, steps, heads, key, value)
    states = torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None
    _launch(device, "ppo_linear_attention_fwd", dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(q, k, v),
            log_decay.data_ptr(), _ptr(carry), _ptr(done), _ptr(lengths), scale, out.data_ptr(), final.data_ptr(),
            _ptr(states), nbytes, batch, steps, heads, kv_heads, key, value)
    return final, out, states


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, carry, done, lengths, scale):
        final, out, states = _forward(q, k, v, log_decay, carry, done, lengths, scale)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, carry, done, lengths, states)
        ctx.scale = scale
        return final, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dfinal, dout):
        q, k, v, log_decay, carry, done, lengths, states = ctx.saved_tensors
        batch, steps, heads, key = q.shape
        kv_heads, value = v.shape[-2:]
        device, dt = q.device, _DTYPES[q.dtype]
        if dout is None:   # (only the final carry was used)
            dout = torch.zeros(value, dtype=q.dtype, device=device).expand(batch, steps, heads, value)
        dout = _rows(dout)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=device) for x in (q, k, v))
        dcarry = torch.empty_like(carry) if carry is not None and ctx.needs_input_grad[4] else None
        nbytes = _lib.load().ppo_linear_attention_bwd_workspace(dt, batch, steps, heads, kv_heads, key, value)
        work = torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None
        _launch(device, "ppo_linear_attention_bwd", dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(),
                _strides(q, k, v, dout), log_decay.data_ptr(), _ptr(carry), _ptr(done), _ptr(lengths), ctx.scale,
                _ptr(dfinal), _ptr(states), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dcarry), _ptr(work),
                nbytes, batch, steps, heads, kv_heads, key, value)
        return dq, dk, dv, None, dcarry, None, None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     carry: torch.Tensor | None = None, done: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None,
                     scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(final carry [batch, heads, key, value] float32, outputs [batch, steps, heads, value]) of

        S_t = exp(log_decay) * (0 where done_t else S_{t-1}) + k_t v_t^T,  o_t = scale * q_t S_t

    with S_{-1} = carry (None: zeros).  q [batch, steps, heads, key], k
    [batch, steps, kv_heads, key], v [batch, steps, kv_heads, value] in any
    strides, float32 or bfloat16; kv_heads divides heads, and heads in a row
    share a key head, whose gradients are their sums.  log_decay: float32
    [heads], at most 0 (-inf: no memory), a fixed schedule without gradient.
    done: bool [batch, steps], the step starts an episode.  lengths: int32
    [batch], steps of each sequence: what follows in q, k, v is not read, and
    its outputs and gradients are zeros.  scale: key ** -0.5 by default.
    Widths up to 128.  A step's infinities and NaN reach the outputs that the
    recurrence gives them to, and no others."""
    _check_attention("linear_attention", q, k, v, log_decay, carry, done, 4)
    if lengths is not None and (lengths.dtype != torch.int32 or tuple(lengths.shape) != (q.shape[0],)):
        raise ValueError(f"lengths must be int32 [{q.shape[0]}], got {lengths.dtype} {tuple(lengths.shape)}")
    _on_device("linear_attention", q, k, v, log_decay, carry, done, lengths)
    key, value = q.shape[-1], v.shape[-1]
    scale = key ** -0.5 if scale is None else float(scale)
    least = 16 // q.element_size()
    if key < least or value < least:   # the kernels read rows 16 bytes at a time
        more_k, more_v = max(least - key, 0), max(least - value, 0)
        q, k, v = pad(q, (0, more_k)), pad(k, (0, more_k)), pad(v, (0, more_v))
        carry = None if carry is None else pad(carry, (0, more_v, 0, more_k))
        carry, out = linear_attention(q, k, v, log_decay, carry, done, lengths, scale)
        return carry[..., :key, :value].contiguous(), out[..., :value].contiguous()
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    carry, done, lengths = (None if x is None else x.contiguous() for x in (carry, done, lengths))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (carry is not None and carry.requires_grad)):
        return _LinearAttention.apply(q, k, v, log_decay, carry, done, lengths, scale)
    return _forward(q, k, v, log_decay, carry, done, lengths, scale)[:2]


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          carry: torch.Tensor, done: torch.Tensor | None = None, scale: float | None = None,
                          out_carry: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(carry, output [batch, heads, value]) of one step of ``linear_attention``:
    q [batch, heads, key], k and v [batch, kv_heads, width], done [batch].  The new
    carry is written to ``out_carry`` where given (``carry`` itself: in place).
    Without gradients: a step that needs them is a sequence of one."""
    _check_attention("linear_attention_step", q, k, v, log_decay, carry, done, 3)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or carry.requires_grad):
        raise ValueError("linear_attention_step has no gradients: use linear_attention on a sequence of one step")
    if out_carry is not None and (out_carry.dtype != torch.float32 or out_carry.shape != carry.shape
                                  or not out_carry.is_contiguous()):
        raise ValueError(f"out_carry must be contiguous float32 {tuple(carry.shape)}")
    device = _on_device("linear_attention_step", q, k, v, log_decay, carry, done, out_carry)
    batch, heads, key = q.shape
    kv_heads, value = v.shape[-2:]
    scale = key ** -0.5 if scale is None else float(scale)
    q, k, v, log_decay, carry = _rows(q), _rows(k), _rows(v), log_decay.contiguous(), carry.contiguous()
    done = None if done is None else done.contiguous()
    if out_carry is None:
        out_carry = torch.empty(carry.shape, dtype=torch.float32, device=device)
    out = torch.empty((batch, heads, value), dtype=q.dtype, device=device)
    _launch(device, "ppo_linear_attention_step", _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(),
            _strides(q, k, v), log_decay.data_ptr(), _ptr(done), carry.data_ptr(), out_carry.data_ptr(),
            out.data_ptr(), scale, batch, heads, kv_heads, key, value)
    return out_carry, out


# ------------------------------------------------------------- norms and rotation
def rotary_frequencies(rotary: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """float64 [rotary / 2] radians a position: base ** (-2 i / rotary)."""
    if rotary < 0 or rotary % 2:
        raise ValueError(f"rotary columns come in pairs, not {rotary}")
    return base ** (-2.0 * torch.arange(rotary // 2, dtype=torch.float64, device=device) / max(1, rotary))


def _norm_forward(q, k, q_scale, k_scale, frequencies, positions, epsilon, interleaved):
    batch, steps, heads, width = q.shape
    device = q.device
    q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
    k_out = torch.empty(k.shape, dtype=q.dtype, device=device)
    _launch(device, "ppo_qk_norm_rotary_fwd", _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), _strides(q, k),
            _ptr(q_scale), _ptr(k_scale), _ptr(frequencies), _ptr(positions), epsilon, interleaved, q_out.data_ptr(),
            k_out.data_ptr(), batch, steps, heads, k.shape[2], width,
            0 if frequencies is None else frequencies.numel())
    return q_out, k_out


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_scale, k_scale, frequencies, positions, epsilon, interleaved):
        ctx.save_for_backward(q, k, q_scale, k_scale, frequencies, positions)
        ctx.options = epsilon, interleaved
        return _norm_forward(q, k, q_scale, k_scale, frequencies, positions, epsilon, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_scale, k_scale, frequencies, positions = ctx.saved_tensors
        epsilon, interleaved = ctx.options
        batch, steps, heads, width = q.shape
        device = q.device
        gq, gk = _rows(gq), _rows(gk)
        dq = torch.empty(q.shape, dtype=q.dtype, device=device)
        dk = torch.empty(k.shape, dtype=q.dtype, device=device)
        dq_scale = None if q_scale is None or not ctx.needs_input_grad[2] else torch.empty_like(q_scale)
        dk_scale = None if k_scale is None or not ctx.needs_input_grad[3] else torch.empty_like(k_scale)
        nbytes = _lib.load().ppo_qk_norm_rotary_bwd_workspace(width)
        work = torch.empty(nbytes // 4, dtype=torch.float32, device=device)
        _launch(device, "ppo_qk_norm_rotary_bwd", _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), gq.data_ptr(),
                gk.data_ptr(), _strides(q, k, gq, gk), _ptr(q_scale), _ptr(k_scale), _ptr(frequencies),
                _ptr(positions), epsilon, interleaved, dq.data_ptr(), dk.data_ptr(), _ptr(dq_scale), _ptr(dk_scale),
                work.data_ptr(), nbytes, batch, steps, heads, k.shape[2], width,
                0 if frequencies is None else frequencies.numel())
        return dq, dk, dq_scale, dk_scale, None, None, None, None


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_scale: torch.Tensor | None = None,
                   k_scale: torch.Tensor | None = None, frequencies: torch.Tensor | None = None,
                   positions: torch.Tensor | None = None, epsilon: float = 1e-6,
                   interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, k): every row of q [batch, steps, heads, width] and k [batch, steps,
    kv_heads, width] (any strides, float32 or bfloat16) divided by its root mean square,
    scaled by q_scale / k_scale (float32 [width], None: ones), then the pairs
    of its first columns turned by position times frequency: columns (i, i +
    P), or interleaved (2 i, 2 i + 1), for the P frequencies (float64 [P],
    radians; None: no rotation).  positions: int32 [batch, steps]; None: the step.
    Widths up to 256.  Gradients reach q, k and the scales."""
    _check_heads("qk_norm_rotary", q, k, None, 4)
    width = q.shape[-1]
    limit = _lib.load().ppo_qk_norm_rotary_max_width()
    if width > limit:
        raise ValueError(f"qk_norm_rotary takes widths up to {limit}, not {width}")
    for name, x in (("q_scale", q_scale), ("k_scale", k_scale)):
        if x is not None and (x.dtype != torch.float32 or tuple(x.shape) != (width,)):
            raise ValueError(f"{name} must be float32 [{width}], got {x.dtype} {tuple(x.shape)}")
    if frequencies is not None:
        if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or 2 * frequencies.numel() > width:
            raise ValueError(f"frequencies must be float64 [up to {width // 2}], got {frequencies.dtype} "
                             f"{tuple(frequencies.shape)}")
        if frequencies.requires_grad:
            raise ValueError("frequencies get no gradient: pass them detached")
        frequencies = frequencies.contiguous() if frequencies.numel() else None
    if positions is not None and (positions.dtype != torch.int32 or positions.shape != q.shape[:2]):
        raise ValueError(f"positions must be int32 {tuple(q.shape[:2])}, got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    _on_device("qk_norm_rotary", q, k, q_scale, k_scale, frequencies, positions)
    q, k = _rows(q), _rows(k)
    q_scale, k_scale, positions = (None if x is None else x.contiguous() for x in (q_scale, k_scale, positions))
    args = (q, k, q_scale, k_scale, frequencies, positions, float(epsilon), int(interleaved))
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, q_scale, k_scale)):
        return _QKNormRotary.apply(*args)
    return _norm_forward(*args)

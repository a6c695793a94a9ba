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

float32 or bfloat16 storage; states, sums and norms are float32, and outputs are
rounded to their type once.  Inside a bfloat16 sequence the pair products and
the states enter matrix products as two bfloat16 pieces (16 bits or more of
their 24), and a state that is neither an output nor leads to one is formed from
terms of two pieces: what these leave, at most 2^-17 of a term each, is small
beside the outputs' rounding of 2^-8.  The step and the final carry keep all 24.
There is no CPU path:
the kernels run on the device the tensors live on, on its current stream, and can
be captured into a graph.  Before a backward pass is captured, drop every eager
autograd graph of the same leaves: such a graph keeps the leaves' gradient nodes
on the stream it was made on, which a capture on another stream must not join.
Forward-mode tangents are refused.

Limits, past which a call is refused: linear_attention 2^21 sequences (batch *
heads), its step 2^23 - 1, both 65536 heads and 2^30 steps; qk_norm_rotary 8192
heads of either operand and 2^31 - 1 rows of steps (batch * steps).
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.nn.functional import pad

from .. import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_MAX_STRIDE = 1 << 23   # of a step, in elements: the kernels count a chunk's bytes in 32 bits


def _no_tangents(name, *tensors):
    """Refuses forward-mode tangents, which a launch would drop: their tensors need not require gradients."""
    if getattr(forward_ad, "_current_level", 0) >= 0:   # (inside a dual level: elsewhere no tensor has one)
        if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
            raise NotImplementedError(f"{name} has no forward-mode derivatives")


def _on_device(name, *tensors):
    """The index of the device that all of them (None aside) are on."""
    _no_tangents(name, *tensors)
    index = tensors[0].get_device()   # (-1: the host)
    for x in tensors:
        if x is not None and x.get_device() != index:
            raise TypeError(f"{name} runs on tensors of one device")
    if index < 0:
        raise TypeError(f"{name} runs on device tensors")
    return index


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # (a build without devices has none)


def _launch(index, name, *args):
    """Calls an entry point on the device's current stream (the device made current where it is not)."""
    if index == torch.cuda.current_device():
        _lib.call(name, _raw_stream(index), *args)
    else:
        with torch.cuda.device(index):
            _lib.call(name, _raw_stream(index), *args)


def _rows(x):
    """x, or a copy where its columns are not side by side."""
    return x.contiguous() if x.stride(-1) != 1 and x.shape[-1] > 1 else x


def _near_rows(x):
    """x, or a copy where its columns are not side by side or its steps too far apart."""
    return x.contiguous() if x.stride(1) > _MAX_STRIDE and x.shape[1] > 1 else _rows(x)


_STRIDES = {n: ctypes.c_int64 * n for n in (6, 9, 12)}


def _strides(*tensors):
    flat = [s for x in tensors for s in x.stride()[:-1]]
    return _STRIDES[len(flat)](*flat)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _check_heads(name, q, k, v, dims):
    dtype, qs, ks = q.dtype, q.shape, k.shape
    if dtype not in _DTYPES:
        raise TypeError(f"{name} stores float32 or bfloat16, not {dtype}")
    if k.dtype != dtype or (v is not None and v.dtype != dtype):
        raise TypeError("q, k and v must share one dtype" if v is not None else "q and k must share one dtype")
    lead = dims - 2
    if (len(qs) != dims or len(ks) != dims or ks[:lead] != qs[:lead] or ks[-1] != qs[-1]
            or (v is not None and (v.dim() != dims or v.shape[:-1] != ks[:-1]))):
        shapes = ", ".join(str(tuple(x.shape)) for x in (q, k, v) if x is not None)
        raise ValueError(f"need q [{'batch, steps' if dims == 4 else 'batch'}, heads, width], k (and v) of the same "
                         f"batch{' and steps' if dims == 4 else ''} with heads that divide q's; got {shapes}")
    return qs, ks


_max_width = 0
_min_widths = {}   # by dtype


def _min_width(dt):
    width = _min_widths.get(dt)
    if width is None:
        width = _min_widths[dt] = _lib.load().ppo_linear_attention_min_width(dt)
    return width


def _check_attention(name, q, k, v, log_decay, carry, done, dims):
    """The sizes (batch, steps or 1, heads, key heads, key and value width)."""
    global _max_width
    _max_width = _max_width or _lib.load().ppo_linear_attention_max_width()
    qs, ks = _check_heads(name, q, k, v, dims)
    batch, heads, kv_heads, key, value = qs[0], qs[-2], ks[-2], qs[-1], v.shape[-1]
    if (kv_heads == 0) != (heads == 0) or (heads and heads % kv_heads):
        raise ValueError(f"{heads} heads do not share {kv_heads} key heads evenly")
    if not (0 < key <= _max_width and 0 < value <= _max_width):
        raise ValueError(f"{name} takes widths from 1 up to {_max_width}, not {key} and {value}")
    if log_decay.dtype != torch.float32 or log_decay.shape != (heads,):
        raise ValueError(f"log_decay must be float32 [{heads}], got {log_decay.dtype} {tuple(log_decay.shape)}")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a fixed schedule: it gets no gradient, pass it detached")
    if carry is not None and (carry.dtype != torch.float32 or carry.shape != (batch, heads, key, value)):
        raise ValueError(f"carry must be float32 {(batch, heads, key, value)}, got {carry.dtype} {tuple(carry.shape)}")
    if done is not None and (done.dtype != torch.bool or done.shape != qs[:dims - 2]):
        raise ValueError(f"done must be bool {tuple(qs[:dims - 2])}, got {done.dtype} {tuple(done.shape)}")
    return batch, qs[1] if dims == 4 else 1, heads, kv_heads, key, value


# --------------------------------------------------------------------- sequences
def _forward(q, k, v, log_decay, carry, done, lengths, scale, sizes):
    batch, steps, heads, kv_heads, key, value = sizes
    dt = _DTYPES[q.dtype]
    out = q.new_empty((batch, steps, heads, value))
    final = log_decay.new_empty((batch, heads, key, value))   # (float32)
    nbytes = _lib.load().ppo_linear_attention_workspace(dt, batch, steps, heads, key, value)
    states = log_decay.new_empty(nbytes // 4) if nbytes else None
    _launch(q.get_device(), "ppo_linear_attention_fwd", dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(q, k, v),
            log_decay.data_ptr(), _ptr(carry), _ptr(done), _ptr(lengths), scale, out.data_ptr(), final.data_ptr(),
            _ptr(states), nbytes, *sizes)
    return final, out, states


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, carry, done, lengths, scale, sizes):
        final, out, states = _forward(q, k, v, log_decay, carry, done, lengths, scale, sizes)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, carry, done, lengths, states)
        ctx.scale, ctx.sizes = scale, sizes
        return final, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dfinal, dout):
        _no_tangents("linear_attention", dfinal, dout)
        q, k, v, log_decay, carry, done, lengths, states = ctx.saved_tensors
        batch, steps, heads, kv_heads, key, value = ctx.sizes
        dt = _DTYPES[q.dtype]
        if dout is None:   # (only the final carry was used)
            dout = q.new_zeros(value).expand(batch, steps, heads, value)
        dout = _near_rows(dout)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dq = q.new_empty((batch, steps, heads, key))
        dk = q.new_empty((batch, steps, kv_heads, key))
        dv = q.new_empty((batch, steps, kv_heads, value))
        dcarry = torch.empty_like(carry) if carry is not None and ctx.needs_input_grad[4] else None
        nbytes = _lib.load().ppo_linear_attention_bwd_workspace(dt, batch, steps, heads, kv_heads, key, value)
        work = log_decay.new_empty(nbytes // 4) if nbytes else None
        _launch(q.get_device(), "ppo_linear_attention_bwd", dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(),
                _strides(q, k, v, dout), log_decay.data_ptr(), _ptr(carry), _ptr(done), _ptr(lengths), ctx.scale,
                _ptr(dfinal), _ptr(states), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dcarry), _ptr(work),
                nbytes, *ctx.sizes)
        return dq, dk, dv, None, dcarry, None, None, None, None


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
    recurrence gives them to, and no others; what the recurrence gives an
    infinity may come out as NaN."""
    sizes = _check_attention("linear_attention", q, k, v, log_decay, carry, done, 4)
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != sizes[:1]):
        raise ValueError(f"lengths must be int32 [{sizes[0]}], got {lengths.dtype} {tuple(lengths.shape)}")
    _on_device("linear_attention", q, k, v, log_decay, carry, done, lengths)
    key, value = sizes[4:]
    scale = key ** -0.5 if scale is None else float(scale)
    least = _min_width(_DTYPES[q.dtype])
    if key < least or value < least:   # the kernels read rows 16 bytes at a time
        more_k, more_v = max(least - key, 0), max(least - value, 0)
        if more_k:   # (padding by nothing copies)
            q, k = pad(q, (0, more_k)), pad(k, (0, more_k))
        if more_v:
            v = pad(v, (0, more_v))
        carry = None if carry is None else pad(carry, (0, more_v, 0, more_k))
        carry, out = linear_attention(q, k, v, log_decay, carry, done, lengths, scale)
        return carry[..., :key, :value].contiguous(), out[..., :value].contiguous()
    args = (_near_rows(q), _near_rows(k), _near_rows(v), log_decay.contiguous(),
            None if carry is None else carry.contiguous(), None if done is None else done.contiguous(),
            None if lengths is None else lengths.contiguous(), scale, sizes)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (carry is not None and carry.requires_grad)):
        return _LinearAttention.apply(*args)
    return _forward(*args)[:2]


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          carry: torch.Tensor, done: torch.Tensor | None = None, scale: float | None = None,
                          out_carry: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(carry, output [batch, heads, value]) of one step of ``linear_attention``:
    q [batch, heads, key], k and v [batch, kv_heads, width], done [batch].  The new
    carry is written to ``out_carry`` where given (``carry`` itself: in place; else apart from it).
    Without gradients: a step that needs them is a sequence of one."""
    batch, _, *sizes = _check_attention("linear_attention_step", q, k, v, log_decay, carry, done, 3)
    heads, kv_heads, key, value = sizes
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or carry.requires_grad):
        raise ValueError("linear_attention_step has no gradients: use linear_attention on a sequence of one step")
    if out_carry is not None and (out_carry.dtype != torch.float32 or out_carry.shape != carry.shape
                                  or not out_carry.is_contiguous() or out_carry.requires_grad):
        raise ValueError(f"out_carry must be contiguous float32 {tuple(carry.shape)} that needs no gradient")
    if out_carry is not None and 0 < abs(out_carry.data_ptr() - carry.data_ptr()) < 4 * carry.numel():
        raise ValueError("out_carry must be carry itself or memory apart from it")
    index = _on_device("linear_attention_step", q, k, v, log_decay, carry, done, out_carry)
    scale = key ** -0.5 if scale is None else float(scale)
    q, k, v, log_decay, carry = _rows(q), _rows(k), _rows(v), log_decay.contiguous(), carry.contiguous()
    done = None if done is None else done.contiguous()
    if out_carry is None:
        out_carry = carry.new_empty((batch, heads, key, value))
    else:
        torch.autograd.graph.increment_version(out_carry)   # (written in place)
    out = q.new_empty((batch, heads, value))
    _launch(index, "ppo_linear_attention_step", _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(),
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
    q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
    _launch(q.get_device(), "ppo_qk_norm_rotary_fwd", _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), _strides(q, k),
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
        _no_tangents("qk_norm_rotary", gq, gk)
        q, k, q_scale, k_scale, frequencies, positions = ctx.saved_tensors
        epsilon, interleaved = ctx.options
        batch, steps, heads, width = q.shape
        gq, gk = _rows(gq), _rows(gk)
        dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
        dq_scale = None if q_scale is None or not ctx.needs_input_grad[2] else torch.empty_like(q_scale)
        dk_scale = None if k_scale is None or not ctx.needs_input_grad[3] else torch.empty_like(k_scale)
        nbytes = _lib.load().ppo_qk_norm_rotary_bwd_workspace(width)
        work = torch.empty(nbytes // 4, dtype=torch.float32, device=q.device)
        _launch(q.get_device(), "ppo_qk_norm_rotary_bwd", _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), gq.data_ptr(),
                gk.data_ptr(), _strides(q, k, gq, gk), _ptr(q_scale), _ptr(k_scale), _ptr(frequencies),
                _ptr(positions), epsilon, interleaved, dq.data_ptr(), dk.data_ptr(), _ptr(dq_scale), _ptr(dk_scale),
                work.data_ptr(), nbytes, batch, steps, heads, k.shape[2], width,
                0 if frequencies is None else frequencies.numel())
        return dq, dk, dq_scale, dk_scale, None, None, None, None


_max_norm_width = 0


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
    global _max_norm_width
    _max_norm_width = _max_norm_width or _lib.load().ppo_qk_norm_rotary_max_width()
    qs, _ = _check_heads("qk_norm_rotary", q, k, None, 4)
    width = qs[3]
    if width > _max_norm_width:
        raise ValueError(f"qk_norm_rotary takes widths up to {_max_norm_width}, not {width}")
    for name, x in (("q_scale", q_scale), ("k_scale", k_scale)):
        if x is not None and (x.dtype != torch.float32 or x.shape != (width,)):
            raise ValueError(f"{name} must be float32 [{width}], got {x.dtype} {tuple(x.shape)}")
    if frequencies is not None:
        if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or 2 * frequencies.numel() > width:
            raise ValueError(f"frequencies must be float64 [up to {width // 2}], got {frequencies.dtype} "
                             f"{tuple(frequencies.shape)}")
        if frequencies.requires_grad:
            raise ValueError("frequencies get no gradient: pass them detached")
        frequencies = frequencies.contiguous() if frequencies.numel() else None
    if positions is not None and (positions.dtype != torch.int32 or positions.shape != qs[:2]):
        raise ValueError(f"positions must be int32 {tuple(qs[:2])}, got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    _on_device("qk_norm_rotary", q, k, q_scale, k_scale, frequencies, positions)
    q, k = _rows(q), _rows(k)
    q_scale, k_scale, positions = (None if x is None else x.contiguous() for x in (q_scale, k_scale, positions))
    args = (q, k, q_scale, k_scale, frequencies, positions, float(epsilon), int(interleaved))
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, q_scale, k_scale)):
        return _QKNormRotary.apply(*args)
    return _norm_forward(*args)

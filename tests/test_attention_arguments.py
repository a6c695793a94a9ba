"""What linear attention and the query / key norms refuse, on the host."""
import ctypes

import pytest
import torch

from boonta_amd import _lib
from boonta_amd.kernels import linear_attention, linear_attention_step, qk_norm_rotary, rotary_frequencies


def operands(B=2, T=3, H=4, G=2, K=8, V=6, dtype=torch.float32):
    return [torch.zeros(B, T, H, K, dtype=dtype), torch.zeros(B, T, G, K, dtype=dtype),
            torch.zeros(B, T, G, V, dtype=dtype), torch.zeros(H)]


def refused(error, match, f, *args, **kw):
    with pytest.raises(error, match=match):
        f(*args, **kw)


def test_linear_attention_refuses_what_it_does_not_take():
    q, k, v, g = operands()
    refused(TypeError, "device", linear_attention, q, k, v, g)
    refused(TypeError, "float32 or bfloat16", linear_attention, q.half(), k.half(), v.half(), g)
    refused(TypeError, "one dtype", linear_attention, q, k.bfloat16(), v, g)
    refused(ValueError, "need q", linear_attention, q[0], k, v, g)
    refused(ValueError, "need q", linear_attention, q, k[:, :2], v, g)
    refused(ValueError, "need q", linear_attention, q, k, v[:, :, :1], g)
    refused(ValueError, "evenly", linear_attention, q[:, :, :3], k, v, g[:3])
    refused(ValueError, "up to 128", linear_attention, *operands(K=129))
    refused(ValueError, "up to 128", linear_attention, *operands(V=129))
    refused(ValueError, "up to 128", linear_attention, *operands(K=0))
    refused(ValueError, "log_decay", linear_attention, q, k, v, g[:2])
    refused(ValueError, "log_decay", linear_attention, q, k, v, g.double())
    refused(ValueError, "fixed schedule", linear_attention, q, k, v, g.clone().requires_grad_())
    refused(ValueError, "carry", linear_attention, q, k, v, g, torch.zeros(2, 2, 8, 6))
    refused(ValueError, "carry", linear_attention, q, k, v, g, torch.zeros(2, 4, 8, 6).bfloat16())
    refused(ValueError, "done", linear_attention, q, k, v, g, done=torch.zeros(2, 4).bool())
    refused(ValueError, "done", linear_attention, q, k, v, g, done=torch.zeros(2, 3))
    refused(ValueError, "lengths", linear_attention, q, k, v, g, lengths=torch.zeros(2, dtype=torch.int64))
    refused(ValueError, "lengths", linear_attention, q, k, v, g, lengths=torch.zeros(3, dtype=torch.int32))


def test_linear_attention_step_refuses_what_it_does_not_take():
    q, k, v, g = operands()
    q, k, v, carry = q[:, 0], k[:, 0], v[:, 0], torch.zeros(2, 4, 8, 6)
    refused(TypeError, "device", linear_attention_step, q, k, v, g, carry)
    refused(ValueError, "need q", linear_attention_step, q[:, None], k, v, g, carry)
    refused(ValueError, "carry", linear_attention_step, q, k, v, g, carry[:1])
    refused(ValueError, "done", linear_attention_step, q, k, v, g, carry, torch.zeros(2, 1).bool())
    refused(ValueError, "no gradients", linear_attention_step, q, k, v, g, carry.clone().requires_grad_())
    refused(ValueError, "out_carry", linear_attention_step, q, k, v, g, carry, out_carry=carry.transpose(2, 3))
    refused(ValueError, "no gradient", linear_attention_step, q, k, v, g, carry, out_carry=carry.clone().requires_grad_())
    whole = torch.zeros(3, 4, 8, 6)
    refused(ValueError, "apart", linear_attention_step, q, k, v, g, whole[:2], out_carry=whole[1:])
    refused(TypeError, "device", linear_attention_step, q, k, v, g, whole[:2], out_carry=whole[:2])


def test_qk_norm_rotary_refuses_what_it_does_not_take():
    q, k, _, _ = operands()
    f = rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (4,) and f[0] == 1
    refused(ValueError, "pairs", rotary_frequencies, 7, device="cpu")
    refused(TypeError, "device", qk_norm_rotary, q, k)
    refused(TypeError, "one dtype", qk_norm_rotary, q, k.bfloat16())
    refused(ValueError, "need q", qk_norm_rotary, q, k[..., :4])
    refused(ValueError, "up to 256", qk_norm_rotary, *operands(K=257)[:2])
    refused(ValueError, "q_scale", qk_norm_rotary, q, k, torch.ones(7))
    refused(ValueError, "k_scale", qk_norm_rotary, q, k, None, torch.ones(8).bfloat16())
    refused(ValueError, "frequencies", qk_norm_rotary, q, k, frequencies=f.float())
    refused(ValueError, "frequencies", qk_norm_rotary, q, k, frequencies=rotary_frequencies(10, device="cpu"))
    refused(ValueError, "no gradient", qk_norm_rotary, q, k, frequencies=f.clone().requires_grad_())
    refused(ValueError, "positions", qk_norm_rotary, q, k, positions=torch.zeros(2, 3, dtype=torch.int64))
    refused(ValueError, "positions", qk_norm_rotary, q, k, positions=torch.zeros(3, dtype=torch.int32))


def test_the_limits_are_those_stated():
    """One past each of the header's limits is refused, and says which."""
    lib = _lib.load()
    st = (ctypes.c_int64 * 12)(*[0] * 12)

    def refusal(f, *args):
        assert f(*args) == -1
        return lib.ppo_last_error().decode()

    def sequences(batch, steps, heads):
        return refusal(lib.ppo_linear_attention_fwd, None, 0, 1, 1, 1, st, 1, None, None, None, 1.0, 1, 1, None, 0, batch,
                       steps, heads, heads, 8, 8)

    def step(batch, heads):
        return refusal(lib.ppo_linear_attention_step, None, 0, 1, 1, 1, st, 1, None, 1, 1, 1, 1.0, batch, heads, heads, 8, 8)

    def norms(batch, steps, heads, kv_heads):
        return refusal(lib.ppo_qk_norm_rotary_fwd, None, 0, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, batch, steps,
                       heads, kv_heads, 8, 0)

    assert "heads above 65536" in sequences(1, 4, 65537) and "steps above 2^30" in sequences(1, (1 << 30) + 1, 1)
    assert f"batch x heads above {1 << 21}" in sequences((1 << 21) + 1, 4, 1)
    assert f"batch x heads above {(1 << 23) - 1}" in step(1 << 23, 1) and "heads above 65536" in step(1, 65537)
    assert "heads above 8192" in norms(1, 1, 8193, 1) and "heads above 8192" in norms(1, 1, 1, 8193)
    assert "batch x steps above" in norms(1 << 16, 1 << 15, 1, 1)
    lib.ppo_clear_error()


def test_forward_mode_tangents_are_refused():
    """A dual tensor does not require gradients, so a plain launch would drop its tangent."""
    from torch.autograd import forward_ad
    q, k, v, g = operands()
    carry = torch.zeros(2, 4, 8, 6)
    first = [q[:, 0], k[:, 0], v[:, 0], g, carry]
    norms = [q, k, torch.ones(8), torch.ones(8), rotary_frequencies(8, device="cpu")]
    with forward_ad.dual_level():
        for f, args in ((linear_attention, [q, k, v, g, carry]), (linear_attention_step, first), (qk_norm_rotary, norms)):
            for i, x in enumerate(args):
                dual = [*args[:i], forward_ad.make_dual(x, torch.ones_like(x)), *args[i + 1:]]
                for grad in (True, False):
                    with torch.set_grad_enabled(grad):
                        refused(NotImplementedError, "forward-mode", f, *dual)
            refused(TypeError, "device", f, *args)
        narrow = operands(K=3, V=2)
        refused(NotImplementedError, "forward-mode", linear_attention,
                forward_ad.make_dual(narrow[0], torch.ones_like(narrow[0])), *narrow[1:])
        refused(NotImplementedError, "forward-mode", linear_attention_step, *first,
                out_carry=forward_ad.make_dual(torch.zeros(2, 4, 8, 6), torch.ones(2, 4, 8, 6)))


def test_forward_mode_tangents_of_cotangents_are_refused(monkeypatch):
    """Their launches stubbed out: what is refused is refused before them."""
    from torch.autograd import forward_ad
    from boonta_amd.kernels import attention
    monkeypatch.setattr(attention, "_on_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda *a: None)
    q, k, v, g = operands()
    calls = ((lambda: linear_attention(q.requires_grad_(), k, v, g), "linear_attention has no forward-mode"),
             (lambda: qk_norm_rotary(q.requires_grad_(), k), "qk_norm_rotary has no forward-mode"))
    for call, match in calls:
        for i in (0, 1):
            with forward_ad.dual_level():
                out = call()[i]
                dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
                refused(NotImplementedError, match, torch.autograd.grad, out, q, dual)


def test_steps_far_apart_are_copied_where_the_kernel_needs_it(monkeypatch):
    """The norms count in 64 bits: theirs stay where they are."""
    from boonta_amd.kernels import attention
    calls = []
    monkeypatch.setattr(attention, "_on_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda index, name, *a: calls.append(a))
    far = torch.zeros((1 << 23) + 64, dtype=torch.bfloat16).as_strided((1, 2, 1, 8), (0, (1 << 23) + 8, 8, 1))
    qk_norm_rotary(far, far)
    assert calls[-1][1:3] == (far.data_ptr(), far.data_ptr())
    linear_attention(far, far, far, torch.zeros(1))
    assert far.data_ptr() not in calls[-1][1:4] and all(s <= 1 << 23 for s in calls[-1][4])


@pytest.mark.parametrize("dtype,least", [(torch.float32, 4), (torch.bfloat16, 8)])
def test_only_operands_of_narrow_heads_are_padded(dtype, least, monkeypatch):
    """The launch gets the other operands as they are."""
    from boonta_amd.kernels import attention
    calls = []
    monkeypatch.setattr(attention, "_on_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda index, name, *a: calls.append(a))
    for K, V in ((least, least), (least, least - 1), (least - 1, least), (1, 1)):
        q, k, v, g = operands(K=K, V=V, dtype=dtype)
        carry, out = linear_attention(q, k, v, g)
        assert carry.shape == (2, 4, K, V) and out.shape == (2, 3, 4, V)
        passed, widths = calls[-1][1:4], calls[-1][-2:]
        assert widths == (max(K, least), max(V, least))
        for x, at, width in ((q, passed[0], K), (k, passed[1], K), (v, passed[2], V)):
            assert (x.data_ptr() == at) == (width >= least)


def test_the_entry_points_refuse_without_launching():
    lib = _lib.load()
    st = (ctypes.c_int64 * 12)(*[0] * 12)
    fwd = lib.ppo_linear_attention_fwd
    sizes = (2, 4, 2, 2, 8, 8)   # batch, steps, heads, key heads, widths

    def forward(dtype=0, q=1, strides=st, decay=1, final=1, work=None, nbytes=0, sizes=sizes):
        return fwd(None, dtype, q, 1, 1, strides, decay, None, None, None, 1.0, 1, final, work, nbytes, *sizes)

    assert forward(dtype=2) == -1
    assert forward(q=None) == -1 and b"null buffer" in lib.ppo_last_error()
    assert forward(strides=None) == -1 and forward(decay=None) == -1 and forward(final=None) == -1
    assert forward(sizes=(2, 4, 3, 2, 8, 8)) == -1 and b"evenly" in lib.ppo_last_error()
    assert forward(sizes=(2, 4, 3, 0, 8, 8)) == -1
    assert forward(sizes=(2, 4, 2, 2, 129, 8)) == -1 and b"outside 4 .. 128" in lib.ppo_last_error()
    assert forward(sizes=(2, 4, 2, 2, 8, 3)) == -1 and forward(dtype=1, sizes=(2, 4, 2, 2, 7, 8)) == -1
    assert forward(sizes=(2, 4, 1 << 17, 1 << 17, 8, 8)) == -1
    near = (ctypes.c_int64 * 12)(0, -8, 0, *[0] * 9)
    assert forward(strides=near) == -1 and b"step stride" in lib.ppo_last_error()
    assert forward(sizes=(-1, 4, 2, 2, 8, 8)) == -1
    assert forward(sizes=(1 << 30, 4, 2, 2, 8, 8)) == -1
    assert forward(sizes=(0, 4, 2, 2, 8, 8)) == 0
    assert forward(sizes=(1 << 21, 4, 2, 2, 8, 8)) == -1 and b"batch x heads" in lib.ppo_last_error()
    assert forward(sizes=(1, (1 << 30) + 1, 2, 2, 8, 8)) == -1 and b"steps" in lib.ppo_last_error()
    far = (ctypes.c_int64 * 12)(0, 1 << 24, 0, *[0] * 9)
    assert forward(strides=far) == -1 and b"step stride" in lib.ppo_last_error()
    assert forward(strides=far, sizes=(0, 1, 2, 2, 8, 8)) == 0
    long = (1, 1 << 16, 2, 2, 8, 8)
    need = lib.ppo_linear_attention_workspace(0, *long[:3], 8, 8)
    assert need > 0 and forward(sizes=long) == -3 and forward(sizes=long, work=1, nbytes=need - 1) == -3
    assert lib.ppo_linear_attention_bwd_workspace(0, 2, 4, 4, 2, 8, 8) == 4 * 2 * 4 * 4 * 16
    assert lib.ppo_linear_attention_bwd_workspace(0, 2, 4, 4, 4, 8, 8) == 0
    bwd = lib.ppo_linear_attention_bwd
    assert bwd(None, 0, 1, 1, 1, None, st, 1, None, None, None, 1.0, None, None, 1, 1, 1, None, None, 0, *sizes) == -1
    assert bwd(None, 0, 1, 1, 1, 1, st, 1, None, None, None, 1.0, None, None, 1, 1, 1, None, None, 0, 2, 4, 4, 2, 8,
               8) == -3
    step = lib.ppo_linear_attention_step
    assert step(None, 0, 1, 1, 1, st, 1, None, None, 1, 1, 1.0, 2, 2, 2, 8, 8) == -1
    assert step(None, 0, 1, 1, 1, st, 1, None, 1, 1, 1, 1.0, 2, 3, 2, 8, 8) == -1
    assert step(None, 0, 1, 1, 1, st, 1, None, 1, 1, 1, 1.0, 1 << 23, 1, 1, 8, 8) == -1
    norm = lib.ppo_qk_norm_rotary_fwd
    assert norm(None, 0, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, 2, 3, 4, 4, 8, 5) == -1   # 5 pairs of 8
    assert norm(None, 0, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, 2, 3, 4, 4, 8, 4) == -1   # no frequencies
    assert norm(None, 0, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, 2, 3, 4, 4, 257, 0) == -1
    assert norm(None, 0, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, 1 << 16, 1 << 15, 4, 4, 8, 0) == -1
    assert norm(None, 0, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, 0, 3, 4, 4, 8, 0) == 0
    assert lib.ppo_qk_norm_rotary_bwd(None, 0, 1, 1, 1, 1, st, None, None, None, None, 1e-6, 0, 1, 1, 1, 1, None, 0, 2,
                                      3, 4, 4, 8, 0) == -3
    lib.ppo_clear_error()

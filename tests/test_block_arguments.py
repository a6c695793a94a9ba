"""What the gated recurrence, the norms around a block and the token log probabilities refuse, on the host."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from boonta_amd import _lib
from boonta_amd.kernels import gated_scan, gated_scan_step, residual_norm, token_log_probs


def refused(error, match, f, *args, **kw):
    with pytest.raises(error, match=match):
        f(*args, **kw)


def gated_operands(B=2, T=3, F=8, dtype=torch.float32):
    return [torch.zeros(B, T, F, dtype=dtype) for _ in range(3)] + [torch.zeros(F)]


def test_gated_scan_refuses_what_it_does_not_take():
    x, i, d, r = gated_operands()
    refused(TypeError, "device", gated_scan, x, i, d, r)
    refused(TypeError, "float32 or bfloat16", gated_scan, x.half(), i.half(), d.half(), r)
    refused(TypeError, "one dtype", gated_scan, x, i.bfloat16(), d, r)
    refused(ValueError, "one shape", gated_scan, x[0], i[0], d[0], r)
    refused(ValueError, "one shape", gated_scan, x, i[:, :2], d, r)
    refused(ValueError, "one shape", gated_scan, x, i, d[..., :1], r)
    refused(ValueError, "rate", gated_scan, x, i, d, r[:4])
    refused(ValueError, "rate", gated_scan, x, i, d, r.double())
    refused(ValueError, "carry", gated_scan, x, i, d, r, torch.zeros(2, 4))
    refused(ValueError, "carry", gated_scan, x, i, d, r, torch.zeros(2, 8).bfloat16())
    refused(ValueError, "done", gated_scan, x, i, d, r, done=torch.zeros(2, 3))
    refused(ValueError, "done", gated_scan, x, i, d, r, done=torch.zeros(2, 4).bool())
    refused(ValueError, "lengths", gated_scan, x, i, d, r, lengths=torch.zeros(2, dtype=torch.int64))
    refused(ValueError, "lengths", gated_scan, x, i, d, r, lengths=torch.zeros(3, dtype=torch.int32))


def test_gated_scan_step_refuses_what_it_does_not_take():
    x, i, d, r = gated_operands()
    x, i, d, carry = x[:, 0], i[:, 0], d[:, 0], torch.zeros(2, 8)
    refused(TypeError, "device", gated_scan_step, x, i, d, r, carry)
    refused(ValueError, "one shape", gated_scan_step, x[:, None], i, d, r, carry)
    refused(ValueError, "carry", gated_scan_step, x, i, d, r, carry[:1])
    refused(ValueError, "done", gated_scan_step, x, i, d, r, carry, torch.zeros(2, 1).bool())
    refused(ValueError, "no gradients", gated_scan_step, x, i, d, r.clone().requires_grad_(), carry)
    refused(ValueError, "no gradients", gated_scan_step, x, i, d, r, carry.clone().requires_grad_())
    refused(ValueError, "out_carry", gated_scan_step, x, i, d, r, carry, out_carry=torch.zeros(8, 2).t())
    refused(ValueError, "no gradient", gated_scan_step, x, i, d, r, carry, out_carry=carry.clone().requires_grad_())
    whole = torch.zeros(3, 8)
    refused(ValueError, "apart", gated_scan_step, x, i, d, r, whole[:2], out_carry=whole[1:])
    refused(TypeError, "device", gated_scan_step, x, i, d, r, whole[:2], out_carry=whole[:2])


def test_residual_norm_refuses_what_it_does_not_take():
    x = torch.zeros(2, 3, 8)
    w = torch.ones(8)
    refused(TypeError, "device", residual_norm, x, x)
    refused(TypeError, "float32 or bfloat16", residual_norm, x.half(), x.half())
    refused(TypeError, "residual", residual_norm, x, x.bfloat16())
    refused(TypeError, "one dtype", residual_norm, x, x, x.bfloat16())
    refused(ValueError, "one shape", residual_norm, x[0], x[0])
    refused(ValueError, "one shape", residual_norm, x, x[:, :2])
    refused(ValueError, "one shape", residual_norm, x, x, x[:, :1])
    refused(ValueError, "up to 8192", residual_norm, torch.zeros(1, 1, 8193), torch.zeros(1, 1, 8193))
    refused(ValueError, "post_scale", residual_norm, x, x, None, w[:7])
    refused(ValueError, "residual_scale", residual_norm, x, x, None, None, w.bfloat16())
    refused(ValueError, "pre_scale", residual_norm, x, x, None, None, None, w[None])
    refused(ValueError, "without post_norm", residual_norm, x, x, None, w, post_norm=False)
    refused(ValueError, "gate_activation", residual_norm, x, x, x, gate_activation="tanh")
    refused(ValueError, "without a gate", residual_norm, x, x, gate_activation="sigmoid")


def test_token_log_probs_refuses_what_it_does_not_take():
    x, t = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64)
    refused(TypeError, "device", token_log_probs, x, t)
    refused(TypeError, "float32 or bfloat16", token_log_probs, x.half(), t)
    refused(TypeError, "int32 or int64", token_log_probs, x, t.float())
    refused(ValueError, "leading shape", token_log_probs, x, t[:, :2])
    refused(ValueError, "leading shape", token_log_probs, x[0, 0], t[0, 0])
    refused(ValueError, "vocabularies", token_log_probs, x[..., :0], t)
    refused(ValueError, "vocabularies", token_log_probs, torch.zeros(1).expand(2, 3, (1 << 24) + 1), t)
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
        refused(ValueError, "temperature", token_log_probs, x, t, None, temperature)
    refused(ValueError, "top", token_log_probs, x, t, top=9)
    refused(ValueError, "top", token_log_probs, x, t, top=-1)
    refused(ValueError, "top", token_log_probs, torch.zeros(2, 3, 40), t, top=33)
    refused(TypeError, "mask", token_log_probs, x, t, torch.zeros(2, 3, 8))
    refused(ValueError, "broadcast", token_log_probs, x, t, torch.ones(2, 3, 4).bool())


def test_forward_mode_tangents_are_refused():
    x, t = torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        refused(NotImplementedError, "forward-mode", token_log_probs, dual, t)
        refused(NotImplementedError, "forward-mode", residual_norm, x, dual)
        refused(NotImplementedError, "forward-mode", gated_scan, x, dual, x, torch.zeros(8))
        refused(NotImplementedError, "forward-mode", gated_scan_step, x[0], dual[0], x[0], torch.zeros(8), torch.zeros(2, 8))


def test_the_limits_are_those_stated():
    """One past each of the header's limits is refused, and says which."""
    lib = _lib.load()
    st = (ctypes.c_int64 * 10)(*[0] * 10)

    def fails(match, name, *args):
        assert getattr(lib, name)(*args) == -1
        assert match in lib.ppo_last_error().decode()

    def gated(dtype, B, T, F, strides=st):
        return ("ppo_gated_scan_fwd", None, dtype, 1, 1, 1, strides, 1, None, None, None, 1, 1, None, None, 0, B, T, F)

    fails("dtype", *gated(2, 1, 1, 1))
    fails("2^21", *gated(0, (1 << 21) + 1, 1, 1))
    fails("2^30", *gated(0, 1, (1 << 30) + 1, 1))
    fails("2^20", *gated(0, 1, 1, (1 << 20) + 1))
    fails("2^29", *gated(0, 1 << 10, 1, (1 << 19) + 1))
    fails("size", *gated(0, -1, 1, 1))
    far = (ctypes.c_int64 * 10)(0, (1 << 23) + 1, *[0] * 8)
    fails("stride", *gated(0, 1, 2, 1, far))
    fails("null", "ppo_gated_scan_fwd", None, 0, None, 1, 1, st, 1, None, None, None, 1, 1, None, None, 0, 1, 1, 1)
    fails("null", "ppo_gated_scan_bwd", None, 0, 1, 1, 1, 1, st, 1, None, None, None, None, 1, 1, 1, None, None, None, 0, 1, 1, 1)
    fails("null", "ppo_gated_scan_step", None, 0, 1, 1, 1, st, 1, None, None, 1, 1, 1, 1)
    assert lib.ppo_gated_scan_bwd(None, 0, 1, 1, 1, 1, st, 1, None, None, 1, None, 1, 1, 1, None, None, None, 0, 1, 1, 1) == -3

    def residual(dtype, stream, B, T, D):
        return ("ppo_residual_norm_fwd", None, dtype, stream, 1, 1, None, st, None, None, None, 1, 0, 1e-6, 1, 1, None, B, T, D)

    fails("dtype", *residual(0, 1, 1, 1, 1))
    fails("width", *residual(0, 0, 1, 1, lib.ppo_residual_norm_max_width() + 1))
    fails("batch x steps", *residual(0, 0, 1 << 16, 1 << 15, 1))
    fails("null", "ppo_residual_norm_fwd", None, 0, 0, None, 1, None, st, None, None, None, 1, 0, 1e-6, 1, 1, None, 1, 1, 1)
    assert lib.ppo_residual_norm_bwd(None, 0, 0, 1, 1, None, 1, 1, st, None, None, None, 1, 0, 1, 1, 1, None, 1, None, None, None,
                                     0, 1, 1, 1) == -3

    def tokens(dtype, T, top, B, S, V):
        return ("ppo_token_log_probs_fwd", None, dtype, 1, 1, 0, None, st, T, top, 1, 1, None, 1, 1, None, 0, B, S, V)

    fails("dtype", *tokens(3, 1.0, 0, 1, 1, 1))
    fails("size", *tokens(0, 1.0, 0, 1, 1, 0))
    fails("size", *tokens(0, 1.0, 0, 1, 1, lib.ppo_token_log_probs_max_vocab() + 1))
    fails("2^24", *tokens(0, 1.0, 0, 1 << 12, 1 << 12, 1))
    fails("temperature", *tokens(0, 0.0, 0, 1, 1, 1))
    fails("alternatives", *tokens(0, 1.0, lib.ppo_token_log_probs_max_top() + 1, 1, 1, 64))
    assert lib.ppo_token_log_probs_fwd(None, 0, 1, 1, 0, None, st, 1.0, 0, 1, 1, None, None, None, None, 0, 1, 1, 1 << 17) == -3
    # nothing to do is no error, whatever the pointers
    assert lib.ppo_gated_scan_fwd(None, 0, None, None, None, None, None, None, None, None, None, None, None, None, 0, 0, 3, 3) == 0
    assert lib.ppo_residual_norm_fwd(None, 0, 0, None, None, None, None, None, None, None, 1, 0, 1e-6, None, None, None, 0, 1, 1) == 0
    assert lib.ppo_token_log_probs_fwd(None, 0, None, None, 0, None, None, 1.0, 0, None, None, None, None, None, None, 0, 0, 1, 1) == 0


def test_workspaces_follow_the_sizes():
    """Sizes of the host-only functions: none where there is no work, float32 states and sums otherwise."""
    lib = _lib.load()
    for f in (lib.ppo_gated_scan_workspace, lib.ppo_gated_scan_states, lib.ppo_gated_scan_bwd_workspace):
        assert f(0, 0, 5, 5) == f(0, 5, 0, 5) == f(0, 5, 5, 0) == 0
    assert lib.ppo_gated_scan_workspace(1, 4096, 100, 256) == 0            # sequences fill the chip: no segments
    assert lib.ppo_gated_scan_workspace(1, 1, 65536, 256) > 0
    assert lib.ppo_gated_scan_states(0, 3, 5, 7) >= 4 * 3 * 7
    assert lib.ppo_gated_scan_bwd_workspace(0, 2, 64, 8) >= 4 * 2 * 8
    assert lib.ppo_residual_norm_bwd_workspace(0, 2, 3, 8) >= 4 * 2 * 8 and lib.ppo_residual_norm_bwd_workspace(0, 0, 3, 8) == 0
    assert lib.ppo_token_log_probs_workspace(4, 1, 1000, 8) == 0 and lib.ppo_token_log_probs_workspace(4, 1, 1 << 17, 8) > 0

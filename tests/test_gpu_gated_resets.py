"""A decay gate of NaN behind a reset of the gated recurrence: the episode before the reset keeps its gradients.

A cotangent passes no reset backward, so that every gradient before it, the carry's too, is bit for bit that of the same
call with ordinary gates: whichever chunk, tile or segment the reset and the bad step fall into."""
import pytest
import torch

from boonta_amd.kernels import gated_scan

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def gradients(leaves, done, cots):
    outs = gated_scan(*leaves, done)
    return outs[1].detach(), torch.autograd.grad(outs, leaves, cots)


# sequences stepped through, of one tile, of several, and in segments
@pytest.mark.parametrize("T,F,dtype", [(6, 24, F32), (60, 24, BF16), (61, 3, F32), (700, 130, BF16), (3000, 24, F32), (9000, 16, BF16)])
def test_a_bad_decay_behind_a_reset_leaves_the_episode_before_it_alone(T, F, dtype):
    gen = torch.Generator().manual_seed(T)
    x, i, d = (torch.randn(2, T, F, generator=gen).to(dtype).cuda().requires_grad_() for _ in range(3))
    rate, carry = torch.rand(F, generator=gen).cuda().requires_grad_(), torch.randn(2, F, generator=gen).cuda().requires_grad_()
    cots = [torch.randn(2, F, generator=gen).cuda(), torch.randn(2, T, F, generator=gen).to(dtype).cuda()]
    feature = F // 2
    for reset in range(0, 6) if T == 6 else (0, *range(T // 2, T // 2 + 8), T - 5):
        done = torch.zeros(2, T, dtype=torch.bool, device="cuda")
        done[1, reset] = True
        out, want = gradients([x, i, d, rate, carry], done, cots)
        for behind in range(min(4, T - reset)):
            bad = d.detach().clone()
            bad[1, reset + behind, feature] = float("nan")
            got_out, got = gradients([x, i, bad.requires_grad_(), rate, carry], done, cots)
            where = (reset, behind)
            assert torch.equal(got_out[:, :reset], out[:, :reset]) and got_out[1, reset + behind, feature].isnan(), where
            for a, b in zip(got[:3], want[:3]):
                assert torch.equal(a[:, :reset], b[:, :reset]), where
                assert torch.equal(a[0], b[0]), where
            assert torch.equal(got[4], want[4]), where

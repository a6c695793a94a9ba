"""Logits that a mask does not allow get no gradient, whatever the cotangents of their row are."""
import pytest
import torch

from boonta_amd.kernels import token_log_probs

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NAN, INF = float("nan"), float("inf")


# backward of several rows' units together, and of a row in parts
@pytest.mark.parametrize("V", [1, 5, 43, 700, 8192, 8193, 20000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_logits_get_none_of_bad_cotangents(V, dtype):
    gen = torch.Generator().manual_seed(V)
    rows = 13
    x = torch.randn(rows, V, generator=gen).to(dtype).cuda().requires_grad_()
    mask = (torch.rand(rows, V, generator=gen) < 0.6).cuda()
    tokens = torch.randint(0, V, (rows,), generator=gen).cuda()
    mask[torch.arange(rows), tokens] = True
    mask[:5] = False                               # ended environments: nothing is allowed
    g, h = torch.randn(2, rows, generator=gen).cuda()
    clean, = torch.autograd.grad(list(token_log_probs(x, tokens, mask)[:2]), x, [g, h])
    h[0], h[1], h[2], g[3], h[4], g[4] = NAN, INF, -INF, NAN, NAN, INF
    h[5], h[6], g[7], g[8], h[11], h[12] = NAN, INF, NAN, -INF, 3e38, -1e35
    grad, = torch.autograd.grad(list(token_log_probs(x, tokens, mask)[:2]), x, [g, h])
    assert not grad[~mask].isnan().any() and not grad[~mask].any() and not grad[:5].any()
    assert torch.equal(grad[9:11], clean[9:11])
    if V > 1:
        assert not grad[5:9][mask[5:9]].isfinite().all()
    # a logit of -inf is one that is not allowed
    same = torch.where(mask, x.detach(), -INF).requires_grad_()
    again, = torch.autograd.grad(list(token_log_probs(same, tokens)[:2]), same, [g, h])
    assert not again[~mask].isnan().any() and not again[~mask].any()

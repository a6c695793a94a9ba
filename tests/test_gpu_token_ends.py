"""Given tokens whose logits are the lowest that their type holds (a mask that a caller has added to them): allowed tokens
like any other, with the log probability of the formula, their gradient and their place among the alternatives.

N = 2^-24.  (x - max) / T is off by four roundings (a difference, the temperature's inverse, its product, the
sum with the row's log sum), which is below 2^-100 of it; past float32's range it is -inf.  A gradient at such a token is g /
T, whose two roundings and p = 0; elsewhere -g p / T, p within 64 roundings (equal logits, exact sums up to the count
of them), and bf16's rounding of 2^-8."""
import math

import numpy as np
import pytest
import torch

from boonta_amd.kernels import token_log_probs
from oracle import tokens as otok

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
N = 2.0 ** -24


# rows of a wave's lanes, of a wave each, of a workgroup, in segments; backward flat and of one row a workgroup
@pytest.mark.parametrize("rows,V", [(3, 2), (5, 43), (9, 300), (2100, 300), (4, 700), (3, 9000), (2, 70000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_token_of_the_lowest_value_is_a_token(rows, V, dtype):
    low = torch.finfo(dtype).min
    x = torch.full((rows, V), low, dtype=dtype, device="cuda")
    x[:, 0] = 1.0
    token = V - 1
    mask = torch.ones(rows, V, dtype=torch.bool, device="cuda")
    mask[0, token] = False                  # the first row's is not allowed
    tokens = torch.full((rows,), token, device="cuda")
    g = torch.linspace(0.5, 1.5, rows, device="cuda")
    for temperature in (0.5, 1.0, 3.0):
        for top in (0, 2):
            leaf = x.clone().requires_grad_()
            out = token_log_probs(leaf, tokens, mask, temperature, top)
            grad, = torch.autograd.grad(out.log_prob, leaf, g)
            host = x.double().cpu().numpy(), tokens.cpu().numpy()
            lp, _ = otok.log_probs(*host, mask.cpu().numpy(), temperature)
            with np.errstate(over="ignore"):
                want = lp.astype(np.float32)
            got = out.log_prob.detach().cpu().numpy()
            assert got[0] == -math.inf and np.isfinite(want[1:]).all() == (temperature >= 1)
            assert (np.isfinite(got) == np.isfinite(want)).all() and (got[~np.isfinite(want)] == -math.inf).all()
            fin = np.isfinite(want)
            assert (np.abs(got[fin].astype(np.float64) - lp[fin]) <= 4 * N * np.abs(lp[fin])).all()
            if top:
                second = 1 if V > 2 else -1
                assert out.top_tokens[1:].tolist() == [[0, 1]] * (rows - 1) and out.top_tokens[0].tolist() == [0, second]
                assert out.top_log_probs[:, 0].abs().max() == 0
                assert (out.top_log_probs[1:, 1].cpu().numpy() == got[1:]).all()
            dlogits = otok.vjp(*host, g.double().cpu().numpy(), np.zeros(rows), mask.cpu().numpy(), temperature)
            tol = (64 * N + (2.0 ** -8 if dtype == BF16 else 0)) * np.abs(dlogits)
            assert dlogits[1:, token].min() > 0 and (np.abs(grad.double().cpu().numpy() - dlogits) <= tol).all()


@pytest.mark.parametrize("V", [43, 700, 9000])
def test_differences_past_the_types_range(V):
    """From 3e38 down to -3e38, which float32 does not hold the difference of: at a temperature of 10 the log probability is -6e37."""
    x = torch.full((2, V), -3e38, device="cuda")
    x[:, 0] = 3e38
    leaf, tokens = x.clone().requires_grad_(), torch.tensor([1, V - 1], device="cuda")
    for temperature, want in ((10.0, -6e37), (1.0, -math.inf)):
        out = token_log_probs(leaf, tokens, None, temperature, 2)
        grad, = torch.autograd.grad(out.log_prob.sum(), leaf)
        for got in (out.log_prob.detach(), out.top_log_probs[:, 1]):
            np.testing.assert_allclose(got.cpu().numpy(), want, rtol=1e-6)
        exp = torch.zeros_like(x)
        exp[:, 0] = -1 / temperature
        exp[torch.arange(2), tokens] = 1 / temperature
        torch.testing.assert_close(grad, exp, rtol=1e-6, atol=0)
        assert not out.entropy.detach().any()

"""Rows of one likely token and many far ones of one logit, whose terms are 0.57 units in the last place of the sum that
they are added to: one after another they would each round up, half a unit too much for every term.

N = 2^-24.  A thread adds the 8 terms of a unit first, and so a sum at most V / 2048 of those one after another, 7 in
each and 11 over lanes and waves: the row's sum is within V / 2048 + 64 roundings, which is what log_prob is off by."""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import token_log_probs
from oracle import tokens as otok

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
N = 2.0 ** -24


# rows of a wave's lanes, of a wave each, of a workgroup, and in segments
@pytest.mark.parametrize("rows,V,top", [(5, 43, 0), (5, 2000, 1), (3000, 8192, 0), (40, 32768, 0), (40, 32768, 3), (600, 50001, 0),
                                        (2, 131072, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_tokens_of_one_logit_are_counted(rows, V, top, dtype):
    x = torch.full((rows, V), -16.5, dtype=dtype, device="cuda")
    x[torch.arange(rows), (torch.arange(rows) * 977) % V] = 0.0
    tokens = ((torch.arange(rows) * 977) % V).cuda()
    out = token_log_probs(x, tokens, None, 1.0, top)
    want, entropy = otok.log_probs(x[:1].double().cpu().numpy(), tokens[:1].cpu().numpy())   # (every row's)
    R = V / 2048 + 64
    assert (np.abs(out.log_prob.double().cpu().numpy() - want) <= (R + 4 * np.abs(want)) * N).all()
    assert (np.abs(out.entropy.double().cpu().numpy() - entropy) <= 2 * (R + 44) * (np.log(V) + 1) * N).all()
    if top:
        assert torch.equal(out.top_tokens[:, 0], tokens) and torch.equal(out.top_log_probs[:, 0], out.log_prob)

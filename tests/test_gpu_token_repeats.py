"""Gradients of logits bit for bit the same in every run, the signs of their zeros too: the last units of rows that 8
does not divide overlap, and both of their threads have to write the same."""
import pytest
import torch

from boonta_amd.kernels import token_log_probs

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("V", [9, 17, 19, 31, 43, 1001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_bits_in_every_run(V, dtype):
    gen = torch.Generator(device="cuda").manual_seed(V)
    rows = 3000000 // V
    x = torch.randn(rows, V, generator=gen, device="cuda").to(dtype).requires_grad_()
    mask = torch.rand(rows, V, generator=gen, device="cuda") < 0.6
    # tokens of the last unit: their thread adds to its columns
    tokens = torch.randint(V - 3, V, (rows,), generator=gen, device="cuda")
    mask.scatter_(1, tokens[:, None], True)
    g, h = torch.randn(2, rows, generator=gen, device="cuda")
    bits = torch.int32 if dtype == F32 else torch.int16

    def run():
        out = token_log_probs(x, tokens, mask)
        return torch.autograd.grad([out.log_prob, out.entropy], x, [g, h])[0].view(bits)

    first = run()
    for _ in range(8):
        assert torch.equal(run(), first)
    # a zero's sign is that of 0 times the row's factor, whichever thread wrote it
    signs = (first < 0) & ~mask
    assert torch.equal(signs.any(1), (signs | mask).all(1) & (~mask).any(1))

"""The norms around a block over more rows than a launch has workgroups, at widths of 3 to 16 waves: values and
gradients within the bounds of tests/test_gpu_residual_norm.py, the scales' among them, and the same twice."""
import pytest
import torch

from test_gpu_residual_norm import BF16, F32, check, problem, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("size", [(3, 700, 1333), (2, 500, 2500), (1, 700, 3001), (1, 600, 4500), (1, 530, 8191)])
def test_rows_past_the_workgroups(size, types):
    ops = problem(sum(size), *size, *types, packed=True)
    gen = torch.Generator().manual_seed(5)
    cots = [torch.randn(size, generator=gen).to(t).cuda() for t in (types[1], types[0])]
    outs, grads = run(ops, True, "sigmoid", cots)
    check(ops, True, "sigmoid", cots, outs, grads)
    again = run(ops, True, "sigmoid", cots)
    assert all(torch.equal(a, b) for a, b in zip((*outs, *grads.values()), (*again[0], *again[1].values())))

"""The query / key norms with rotation (forward and backward) against the float64 oracle
(oracle/attention.py).

Tolerances: float32 arithmetic loses at most ROUNDS = D / 8 + 24 roundings of
2^-24 relative to the sizes of an output's terms (|y| of both columns of a
pair; the row's largest |e| for gradients, whose mean runs over the row); the
angle is formed in float64 and its float32 sine and cosine are within 2^-22.
bf16 storage adds the output's own rounding, 2^-8 of its value.  dscale sums N
rows in float32: sqrt is not assumed, N / 64 + D roundings of the sum of |terms|."""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import qk_norm_rotary, rotary_frequencies
from oracle import attention as oat

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def np64(x):
    return x.detach().double().cpu().numpy()


def problem(seed, B, T, H, G, D, dtype, packed, far):
    gen = torch.Generator().manual_seed(seed)
    if packed:
        whole = torch.randn(B, T, (H + G) * D + 5, generator=gen).to(dtype).cuda()
        q = whole[..., 3:3 + H * D].unflatten(-1, (H, D))
        k = whole[..., 3 + H * D:3 + (H + G) * D].unflatten(-1, (G, D))
    else:
        q, k = (torch.randn(B, T, h, D, generator=gen).to(dtype).cuda() for h in (H, G))
    scales = [(1 + 0.2 * torch.randn(D, generator=gen)).cuda() for _ in range(2)]
    positions = torch.randint(0, 1 << 30 if far else 100, (B, T), generator=gen, dtype=torch.int32).cuda()
    return q, k, scales, positions


CASES = [  # batch, steps, heads, key heads, width, rotary
    (1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 2, 2), (2, 3, 2, 1, 7, 4), (3, 5, 4, 2, 16, 16), (2, 33, 3, 1, 20, 20), (1, 70, 6, 2, 75, 40),
    (2, 40, 8, 8, 64, 64), (2, 17, 4, 4, 128, 64), (1, 19, 2, 2, 128, 128), (3, 11, 5, 1, 100, 100), (2, 9, 2, 1, 256, 256),
    (1, 5, 2, 1, 255, 254), (1, 3, 40, 7, 48, 32),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_norms_and_rotation_match_the_definition(case, interleaved, dtype):
    B, T, H, G, D, R = case
    for packed, far in ((False, False), (True, True)):
        q, k, scales, positions = problem(sum(case), B, T, H, G, D, dtype, packed, far)
        f = rotary_frequencies(R)
        leaves = [x.detach().requires_grad_() for x in (q, k, *scales)]
        outs = qk_norm_rotary(*leaves, f, positions, 1e-6, interleaved)
        gen = torch.Generator().manual_seed(1)
        cots = [torch.randn(x.shape, generator=gen).to(dtype).cuda() for x in (q, k)]
        grads = torch.autograd.grad(outs, leaves, cots)
        rounds = (D / 8 + 24) * 2.0 ** -24
        for i, x in enumerate((q, k)):
            n, w, c = np64(x), np64(scales[i]), np64(cots[i])
            want = oat.norm_rotary(n, w, np64(f), positions.cpu().numpy(), 1e-6, interleaved)
            size = np.abs(want).max(-1, keepdims=True)
            tol = rounds * size + (2.0 ** -8 * np.abs(want) if dtype == BF16 else 0)
            assert outs[i].dtype == dtype and (np.abs(np64(outs[i]) - want) <= tol).all()
            dx, dscale = oat.norm_rotary_vjp(n, w, np64(f), positions.cpu().numpy(), 1e-6, interleaved, c)
            rstd = 1 / np.sqrt((n * n).mean(-1, keepdims=True) + 1e-6)
            size = rstd * (np.abs(c).max(-1, keepdims=True) * 2 * np.abs(w).max() * (1 + np.abs(n * rstd).max(-1, keepdims=True)))
            tol = rounds * size + (2.0 ** -8 * np.abs(dx) if dtype == BF16 else 0)
            assert (np.abs(np64(grads[i]) - dx) <= tol).all()
            terms = (2 * np.abs(c).max(-1, keepdims=True) * np.abs(n * rstd)).reshape(-1, D).sum(0)
            rows = n.size / D
            assert (np.abs(np64(grads[2 + i]) - dscale) <= (rows / 64 + D + 24) * 2.0 ** -24 * terms).all()


def test_without_scales_positions_or_rotation():
    q, k, scales, _ = problem(3, 2, 9, 2, 1, 24, F32, False, False)
    a = qk_norm_rotary(q, k)
    want = np64(q) / np.sqrt((np64(q) ** 2).mean(-1, keepdims=True) + 1e-6)
    np.testing.assert_allclose(np64(a[0]), want, rtol=3e-6)
    f = rotary_frequencies(24)
    steps = torch.arange(9, dtype=torch.int32, device="cuda").expand(2, 9)
    for x, y in zip(qk_norm_rotary(q, k, *scales, f), qk_norm_rotary(q, k, *scales, f, steps)):
        assert torch.equal(x, y)
    leaves = [q.requires_grad_(), k.requires_grad_()]
    g = torch.autograd.grad(qk_norm_rotary(q, k, None, None, f)[0].sum(), leaves)
    assert not g[1].any() and g[0].any()


def test_empty_batches_and_rows_of_zeros():
    for B, T, H in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        q, k, scales, _ = problem(4, B, T, H, H, 8, BF16, False, False)
        leaves = [x.requires_grad_() for x in (q, k, *scales)]
        out = qk_norm_rotary(*leaves)
        grads = torch.autograd.grad(out, leaves, [torch.ones_like(x) for x in out])
        assert out[0].shape == q.shape and not grads[2].any() and not grads[3].any()
    q = torch.zeros(1, 2, 1, 64, device="cuda").requires_grad_()
    out = qk_norm_rotary(q, q.detach(), frequencies=rotary_frequencies(64))[0]
    assert not out.any() and torch.isfinite(torch.autograd.grad(out.sum(), q)[0]).all()


def test_a_bad_row_stays_alone():
    q, k, scales, positions = problem(5, 2, 30, 3, 1, 64, BF16, False, False)
    want = qk_norm_rotary(q, k, *scales, rotary_frequencies(64), positions)
    q[1, 7, 2, 5] = float("nan")
    got = qk_norm_rotary(q, k, *scales, rotary_frequencies(64), positions)
    assert got[0][1, 7, 2].isnan().all() and torch.equal(got[1], want[1])
    got[0][1, 7, 2] = want[0][1, 7, 2]
    assert torch.equal(got[0], want[0])


def test_many_rows_and_the_same_twice():
    """More tiles than the backward pass has workgroups."""
    q, k, scales, positions = problem(6, 40, 700, 3, 1, 64, BF16, True, False)
    leaves = [x.detach().requires_grad_() for x in (q, k, *scales)]
    f = rotary_frequencies(64)
    runs = []
    for _ in range(2):
        outs = qk_norm_rotary(*leaves, f, positions)
        runs.append((*outs, *torch.autograd.grad(outs, leaves, [x.detach() * 0.5 + 0.25 for x in outs])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    for i, x in enumerate((q, k)):
        c = np64(outs[i].detach() * 0.5 + 0.25)
        dx, dscale = oat.norm_rotary_vjp(np64(x), np64(scales[i]), np64(f), positions.cpu().numpy(), 1e-6, False, c)
        assert np.linalg.norm(np64(runs[0][2 + i]) - dx) <= 2.0 ** -8 * np.linalg.norm(dx)
        assert np.linalg.norm(np64(runs[0][4 + i]) - dscale) <= 2e-6 * np.linalg.norm(dscale)


def test_thousands_of_heads_shared_by_many_steps():
    """8191 key heads beside one query head, the keys' step stride zero: every
    step's row of each head is that head's, whatever the rows of a tile."""
    T, G = 66 * 4096, 8191
    gen = torch.Generator().manual_seed(8)
    q = torch.randn(1, T, 1, 1, generator=gen).to(BF16).cuda()
    k = torch.randn(1, 1, G, 1, generator=gen).to(BF16).cuda()
    want = (k.float() / (k.float().square() + 1e-6).sqrt())[0, 0]
    q_out, k_out = qk_norm_rotary(q, k.expand(1, T, G, 1))
    assert (k_out[0] == k_out[0, :1]).all()
    assert ((k_out[0, 0].float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20).all()
    assert ((q_out[..., 0] > 0) == (q[..., 0] > 0)).all()


def test_a_captured_pass_replays():
    sets = [problem(7 + i, 2, 50, 2, 1, 32, F32, False, False) for i in range(3)]
    f = rotary_frequencies(32)

    def run(q, k, scales, positions):
        outs = qk_norm_rotary(q, k, *scales, f, positions)
        return (*outs, *torch.autograd.grad(outs, [q, k, *scales], [torch.ones_like(x) for x in outs]))

    want = []
    for q, k, scales, positions in sets:
        ready = [x.detach().clone().requires_grad_() for x in (q, k, *scales)]
        want.append([x.detach() for x in run(ready[0], ready[1], ready[2:], positions)])
    q, k, s0, s1 = [x.detach().clone().requires_grad_() for x in (sets[0][0], sets[0][1], *sets[0][2])]
    positions = sets[0][3].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(q, k, [s0, s1], positions)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(q, k, [s0, s1], positions)
    for i in (1, 2, 0):
        with torch.no_grad():
            for x, y in zip((q, k, s0, s1, positions), (sets[i][0], sets[i][1], *sets[i][2], sets[i][3])):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def test_steps_far_apart():
    """A time-major batch wider than 2^23 elements a step, read where it is, forward and backward."""
    wide = torch.randn((2 << 23) + 512, generator=torch.Generator().manual_seed(9)).to(BF16).cuda()
    q = wide.as_strided((1, 3, 2, 64), (0, (1 << 23) + 64, 64, 1)).requires_grad_()
    near = q.detach().clone().contiguous().requires_grad_()
    assert q.stride(1) > 1 << 23 and near.is_contiguous()
    cot = wide.as_strided((1, 3, 2, 64), (0, (1 << 23) + 128, 64, 1))
    f = rotary_frequencies(64)
    a, b = (qk_norm_rotary(x, x.detach(), frequencies=f) for x in (q, near))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(*(torch.autograd.grad(x, y, cot)[0] for x, y in ((a[0], q), (b[0], near))))

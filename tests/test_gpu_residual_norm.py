"""The norms around a block (forward and backward) against the float64 oracle (oracle/residual.py).

Tolerances.  A row's float32 sum of squares takes at most 8 + 6 + 16 additions of
positive terms, so 1 / rms is within 20 roundings of 2^-24; with the products
and the sigmoid (argument up to 8: 12 more) n and the gate are within R = 40, and
y within R A, A = |x| + |scale gate n|.  Where y's terms cancel, the relative
error of its rms grows by k = rms(A) / rms(y), so z and the gradients are within
R' (1 + k) of the sizes of their terms, R' = 128 with their own sums and
products; sizes are the rows' largest.  bf16 storage adds its rounding, 2^-8 of
the value.  A scale's gradient sums `rows` terms: rows / 8 + 64 roundings more
of the sum of their sizes."""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import residual_norm
from oracle import residual as ores

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("block", "residual", "gate", "post", "scale", "pre")
HALF = 2.0 ** -24


def np64(x):
    return x.detach().double().cpu().numpy()


def problem(seed, B, T, D, dtype, stream, gate=True, post=True, packed=False):
    gen = torch.Generator().manual_seed(seed)
    if packed:
        whole = torch.randn(T, B, 2 * D + 5, generator=gen).to(dtype).cuda().transpose(0, 1)
        u, g = whole[..., 1:1 + D], whole[..., 2 + D:2 + 2 * D]
        x = torch.randn(B, T, D + 3, generator=gen).to(stream).cuda()[..., 2:2 + D]
    else:
        u, g = (torch.randn(B, T, D, generator=gen).to(dtype).cuda() for _ in range(2))
        x = torch.randn(B, T, D, generator=gen).to(stream).cuda()
    scales = [(1 + 0.3 * torch.randn(D, generator=gen)).cuda() for _ in range(3)]
    return dict(block=u, residual=x, gate=g if gate else None, post=scales[0] if post else None, scale=scales[1],
                pre=scales[2])


def call(ops, post_norm, activation, epsilon=1e-6):
    return residual_norm(ops["block"], ops["residual"], ops["gate"], ops["post"], ops["scale"], ops["pre"],
                         post_norm=post_norm, gate_activation=activation, epsilon=epsilon)


def leaves_of(ops):
    return {n: None if x is None else x.detach().requires_grad_() for n, x in ops.items()}


def check(ops, post_norm, activation, cots, outs, grads):
    """cots, outs: (stream, normed); grads by name."""
    D = ops["block"].shape[-1]
    ones = np.ones(D)
    args = [None if ops[n] is None else np64(ops[n]) for n in NAMES[:3]]
    args += [ones if ops[n] is None else np64(ops[n]) for n in NAMES[3:]]
    tail = (post_norm, activation == "sigmoid", 1e-6)
    p = ores.parts(*args, *tail)
    post, scale, pre = args[3:]
    wants = ores.residual_norm(*args, *tail)
    A = np.abs(args[1]) + np.abs(scale * p["gate"] * p["n"])
    k = np.sqrt((A * A).mean(-1, keepdims=True)) * p["ry"]

    def within(got, want, tol):
        tol = tol + (2.0 ** -8 * np.abs(want) if got.dtype == BF16 else 0)
        assert got.shape == want.shape and (np.abs(np64(got) - want) <= tol).all()

    def top(v):
        return np.abs(v).max(-1, keepdims=True)

    within(outs[0], wants[0], 40 * HALF * A)
    within(outs[1], wants[1], 128 * HALF * np.abs(pre) * p["ry"] * (A + np.abs(p["y"]) * k))
    if grads is None:
        return
    dy, dz = (np.zeros_like(A) if c is None else np64(c) for c in cots)
    want = ores.residual_norm_vjp(*args, *tail, dy, dz)
    r = 128 * HALF * (1 + k)
    M = top(dy) + p["ry"] * top(dz * pre) * (1 + top(p["yn"]))
    q = scale * p["gate"]
    sizes = dict(residual=M, block=p["ru"] * M * top(q * post) * (1 + top(p["un"])), gate=M * top(scale) * top(p["n"]))
    for n, x in grads.items():
        assert x.dtype == ops[n].dtype
        if n in sizes:
            within(x, want[n], r * sizes[n])
    rows = A.size / D
    terms = dict(post=M * np.abs(q * p["un"]), scale=M * np.abs(p["gate"] * p["n"]), pre=np.abs(dz) * (np.abs(p["yn"]) + p["ry"] * A))
    for n, t in terms.items():
        if n in grads:
            tol = ((r + (rows / 8 + 64) * HALF) * t).reshape(-1, D).sum(0)
            within(grads[n], want[n], tol)


def run(ops, post_norm, activation, cots):
    leaves = leaves_of(ops)
    outs = call(leaves, post_norm, activation)
    names = [n for n in NAMES if leaves[n] is not None]
    return outs, dict(zip(names, torch.autograd.grad(outs, [leaves[n] for n in names], list(cots))))


WIDTHS = [(1, 1, 1), (2, 3, 2), (3, 5, 7), (1, 9, 8), (2, 33, 20), (5, 13, 64), (2, 40, 333), (1, 70, 512), (2, 3, 513),
          (3, 5, 640), (1, 7, 1333), (2, 3, 2048), (1, 3, 4100), (1, 2, 8191), (1, 3, 8192)]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("size", WIDTHS)
def test_norms_match_the_definition(size, types):
    for i, (gate, post_norm, activation, packed) in enumerate(((True, True, "sigmoid", False), (False, True, None, True),
                                                               (True, False, None, True))):
        ops = problem(sum(size) + i, *size, *types, gate=gate, post=post_norm, packed=packed)
        gen = torch.Generator().manual_seed(9)
        cots = [torch.randn(size, generator=gen).to(t).cuda() for t in (types[1], types[0])]
        outs, grads = run(ops, post_norm, activation, cots)
        assert outs[0].dtype == types[1] and outs[1].dtype == types[0]
        check(ops, post_norm, activation, cots, outs, grads)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(call(ops, post_norm, activation), outs))


def test_without_scales_and_with_one_output_used():
    ops = dict(problem(1, 2, 9, 24, F32, F32, gate=False), post=None, scale=None, pre=None)
    for used in (0, 1):
        leaves = leaves_of(ops)
        outs = call(leaves, True, None)
        cots = [None, None]
        cots[used] = torch.randn(2, 9, 24, generator=torch.Generator().manual_seed(2)).cuda()
        grads = torch.autograd.grad(outs[used], [leaves["block"], leaves["residual"]], cots[used])
        check(ops, True, None, cots, outs, dict(zip(NAMES, grads)))


def test_some_operands_need_no_gradient():
    ops = problem(2, 2, 9, 600, BF16, F32)
    cots = [torch.randn(2, 9, 600).to(t).cuda() for t in (F32, BF16)]
    _, want = run(ops, True, "sigmoid", cots)
    for names in (["residual"], ["gate"], ["pre"], ["block", "scale"]):
        leaves = {n: x.detach().requires_grad_(n in names) for n, x in ops.items()}
        outs = call(leaves, True, "sigmoid")
        got = torch.autograd.grad(outs, [leaves[n] for n in names], cots)
        assert all(torch.equal(a, want[n]) for a, n in zip(got, names))


def test_shared_rows_and_strided_cotangents():
    """A gate shared by a sequence's steps (its gradient their sum), cotangents of other strides, columns not side by side."""
    ops = problem(3, 3, 8, 40, F32, F32)
    shared = ops["gate"][:, :1].clone()
    cots = [torch.randn(8, 3, 40, generator=torch.Generator().manual_seed(i)).cuda().transpose(0, 1) for i in range(2)]
    full = dict(ops, gate=shared.expand(3, 8, 40).contiguous())
    outs, grads = run(full, True, "sigmoid", cots)
    leaf = shared.requires_grad_()
    apart = dict(ops, gate=leaf.expand(3, 8, 40), block=ops["block"].transpose(1, 2).contiguous().transpose(1, 2))
    got = call(apart, True, "sigmoid")
    assert all(torch.equal(a, b) for a, b in zip(got, outs))
    dgate, = torch.autograd.grad(got, leaf, cots)
    torch.testing.assert_close(dgate, grads["gate"].sum(1, keepdim=True), rtol=1e-5, atol=1e-5)


def test_empty_batches_and_rows_of_zeros():
    for B, T in ((0, 3), (2, 0)):
        ops = problem(4, B, T, 24, BF16, F32)
        outs, grads = run(ops, True, None, [torch.empty(B, T, 24, device="cuda"), torch.empty(B, T, 24, device="cuda", dtype=BF16)])
        assert outs[0].shape == (B, T, 24) and not any(grads[n].any() for n in ("post", "scale", "pre"))
    ops = {n: torch.zeros_like(x) if x is not None and x.dim() == 3 else x for n, x in problem(4, 1, 2, 64, F32, F32).items()}
    outs, grads = run(ops, True, None, [torch.ones(1, 2, 64, device="cuda")] * 2)
    assert not outs[0].any() and not outs[1].any() and all(torch.isfinite(x).all() for x in grads.values())


@pytest.mark.parametrize("D", [64, 700])
def test_a_bad_row_stays_alone(D):
    ops = problem(5, 2, 30, D, BF16, BF16)
    cots = [torch.randn(2, 30, D).to(BF16).cuda() for _ in range(2)]
    want_outs, want = run(ops, True, "sigmoid", cots)
    ops["block"][1, 7, 5] = float("nan")
    outs, grads = run(ops, True, "sigmoid", cots)
    for a, b in ((outs[0], want_outs[0]), (outs[1], want_outs[1]), *((grads[n], want[n]) for n in NAMES[:3])):
        a = a.detach().clone()
        assert a[1, 7].isnan().any()
        a[1, 7] = b[1, 7]
        assert torch.equal(a, b)


@pytest.mark.parametrize("size", [(40, 700, 20), (3, 3001, 640)])
def test_many_rows_and_the_same_twice(size):
    """More rows than the launches have places for."""
    ops = problem(6, *size, BF16, BF16, packed=True)
    gen = torch.Generator().manual_seed(3)
    cots = [torch.randn(size, generator=gen).to(BF16).cuda() for _ in range(2)]
    outs, grads = run(ops, True, "sigmoid", cots)
    again, grads2 = run(ops, True, "sigmoid", cots)
    assert all(torch.equal(a, b) for a, b in zip((*outs, *grads.values()), (*again, *grads2.values())))
    check(ops, True, "sigmoid", cots, outs, grads)


def test_a_captured_pass_replays():
    size = (2, 50, 1100)
    sets = [problem(7 + i, *size, BF16, F32) for i in range(3)]
    cots = [torch.randn(size).to(t).cuda() for t in (F32, BF16)]
    want = []
    for ops in sets:
        outs, grads = run(ops, True, "sigmoid", cots)
        want.append([x.detach().clone() for x in (*outs, *grads.values())])
        del outs, grads
    leaves = leaves_of({n: x.clone() for n, x in sets[0].items()})

    def both():
        outs = call(leaves, True, "sigmoid")
        return (*outs, *torch.autograd.grad(outs, list(leaves.values()), cots))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            for n, x in leaves.items():
                x.copy_(sets[i][n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def test_on_another_stream():
    ops = problem(11, 4, 100, 300, F32, F32)
    want = call(ops, True, None)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = call(ops, True, None)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_past_32_bit_offsets():
    """A stream of over 2^31 elements a step's stride apart, read where it is."""
    far = (1 << 31) // 2 + 64
    wide = torch.zeros(2 * far + 256, dtype=BF16, device="cuda")
    x = wide.as_strided((1, 3, 64), (0, far, 1))
    near = torch.randn(1, 3, 64, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    x.copy_(near)
    u = torch.randn(1, 3, 64, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    assert x.stride(1) * 2 > 1 << 31
    assert all(torch.equal(a, b) for a, b in zip(residual_norm(u, x), residual_norm(u, near)))

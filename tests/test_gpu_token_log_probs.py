"""Token log probabilities, entropies, top alternatives and gradients against the float64 oracle (oracle/tokens.py).

Tolerances, N = 2^-24.  An exponent w = (x - max) log2(e) / T takes three roundings,
so e^w is within (3 |w| + 2) N; exponents below -40 count under 2^-40.  A sum adds
at most V / 2048 + 11 terms of one sign after another, each rescaling once more:
S is within R = V / 2048 + 64 roundings (the mean |w| under p is below 40).  log_prob
is within R + 4 |log_prob| roundings, the entropy within R + 44 of its two terms,
ln S and the mean |w|, each at most ln V + 1; a gradient within (R + 60) N of
(|g| + |h| (ln V + 41)) p / T (|log p| of terms that count is below 40), and
4 N |g| / T at the token.  bf16 gradients add their rounding, 2^-8 of the value,
and what falls below the type's normal range, 2^-133.  Tokens are exact."""
import numpy as np
import pytest
import torch

from boonta_amd.kernels import token_log_probs
from oracle import tokens as otok

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
N = 2.0 ** -24


def np64(x):
    return x.detach().double().cpu().numpy()


def problem(seed, lead, V, dtype, mask="rows", spread=2.5, tokens=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(*lead, V, generator=gen)).to(dtype).cuda()
    t = torch.randint(-1, V, lead, generator=gen).to(tokens).cuda()
    m = None
    if mask == "rows":
        m = (torch.rand(*lead, V, generator=gen) < 0.6).cuda()
        m.view(-1, V)[::7] = False     # rows that allow nothing
    elif mask == "one":
        m = (torch.rand(V, generator=gen) < 0.8).cuda()
    g, h = torch.randn(2, *lead, generator=gen).cuda()
    return x, t, m, g, h


def full(mask, x):
    return None if mask is None else mask.expand(x.shape).cpu().numpy()


def check(x, tokens, mask, temperature, out, top=0, grad=None, g=None, h=None):
    V, m, t = x.shape[-1], full(mask, x), tokens.cpu().numpy()
    lp, H = otok.log_probs(np64(x), t, m, temperature)
    R, big = V / 2048 + 64, np.log(V) + 1
    assert out.log_prob.dtype == out.entropy.dtype == F32
    got, fin = np64(out.log_prob), np.isfinite(lp)
    assert (got[~fin] == lp[~fin]).all() and (np.abs(got[fin] - lp[fin]) <= (R + 4 * np.abs(lp[fin])) * N).all()
    assert (np.abs(np64(out.entropy) - H) <= 2 * (R + 44) * big * N).all()
    if top:
        best, which = otok.top(np64(x), top, m, temperature)
        assert out.top_tokens.dtype == tokens.dtype and (out.top_tokens.cpu().numpy() == which).all()
        fin = np.isfinite(best)
        got = np64(out.top_log_probs)
        assert (got[~fin] == -np.inf).all() and (np.abs(got[fin] - best[fin]) <= (R + 4 * np.abs(best[fin])) * N).all()
    if grad is not None:
        g, h = np64(g), np64(h)
        want = otok.vjp(np64(x), t, g, h, m, temperature)
        p = np.exp(otok.log_softmax(otok.masked(np64(x), m), temperature)[0])
        size = (np.abs(g) + np.abs(h) * (np.log(V) + 41))[..., None] * (p + 2.0 ** -40 * (p > 0)) / temperature
        inside = (t >= 0) & (t < V)
        hot = (np.arange(V) == t[..., None]) & inside[..., None]
        tol = (R + 60) * N * size + 4 * N * np.abs(g)[..., None] * hot / temperature
        tol = tol + (2.0 ** -8 * np.abs(want) + 2.0 ** -133 if grad.dtype == BF16 else 2.0 ** -140)
        assert grad.dtype == x.dtype and (np.abs(np64(grad) - want) <= tol).all()
        if m is not None:
            assert not np64(grad)[~m].any()


def run(x, tokens, mask, temperature, top, g, h):
    leaf = x.detach().requires_grad_()
    out = token_log_probs(leaf, tokens, mask, temperature, top)
    return out, torch.autograd.grad([out.log_prob, out.entropy], leaf, [g, h])[0]


VOCABS = [1, 2, 3, 7, 8, 9, 16, 43, 64, 65, 127, 300, 511, 512, 513, 2047, 2049, 5000, 50001, 65537]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", VOCABS)
def test_results_match_the_definition(V, dtype):
    for i, (lead, mask, T, top) in enumerate((((3, 5), "rows", 1.0, min(V, 5)), ((17,), "one", 0.7, 0), ((2, 3), None, 1.3, min(V, 32)))):
        x, t, m, g, h = problem(V + i, lead, V, dtype, mask, tokens=torch.int32 if i else torch.int64)
        out, grad = run(x, t, m, T, top, g, h)
        assert out.log_prob.shape == lead and (out.top_tokens is None) == (top == 0)
        check(x, t, m, T, out, top, grad, g, h)
        with torch.no_grad():
            again = token_log_probs(x, t, m, T, top)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("rows,V", [(1, 131072), (3, 262145), (40, 100003), (1100, 4097)])
def test_rows_in_segments_and_many_rows(rows, V):
    x, t, m, g, h = problem(rows, (rows,), V, BF16, "one")
    out, grad = run(x, t, m, 0.9, 20, g, h)
    check(x, t, m, 0.9, out, 20, grad, g, h)


@pytest.mark.parametrize("rows,V,dtype,mask", [(70, 1030, F32, "rows"), (3000, 1025, BF16, None), (9001, 257, F32, "rows"),
                                               (2047, 2049, BF16, "rows"), (2048, 2049, BF16, "rows"),
                                               (2050, 4100, F32, None), (2049, 8192, BF16, "one"), (2049, 8193, BF16, None)])
def test_many_rows_without_alternatives(rows, V, dtype, mask):
    x, t, m, g, h = problem(rows + V, (rows,), V, dtype, mask)
    out, grad = run(x, t, m, 1.1, 0, g, h)
    check(x, t, m, 1.1, out, 0, grad, g, h)


@pytest.mark.parametrize("rows,V,top,dtype", [(2048, 1025, 32, F32), (2100, 2048, 7, BF16), (2047, 2047, 5, BF16),
                                              (30, 1999, 4, F32), (30, 1030, 1, BF16), (70, 5, 5, F32), (70, 9, 9, BF16)])
def test_many_rows_with_alternatives(rows, V, top, dtype):
    """Rounded to 8ths, so that many are equal; the last rows' are all one value, or not allowed but for one."""
    x, t, m, g, h = problem(rows + top, (rows,), V, dtype)
    x = (8 * x).round() / 8
    x[-3:] = 1.5
    m[-1] = False
    m[-1, V - 1] = True
    out, grad = run(x, t, m, 0.8, top, g, h)
    check(x, t, m, 0.8, out, top, grad, g, h)


@pytest.mark.parametrize("V", [40, 300, 3000, 70000])
def test_equal_values_go_to_the_lowest_index(V):
    gen = torch.Generator().manual_seed(V)
    rows = [torch.zeros(V), torch.randint(0, 3, (V,), generator=gen).float(), torch.arange(V) % 17, -torch.arange(V).float(),
            torch.arange(V).float() / 8, torch.where(torch.rand(V, generator=gen) < 0.5, 0.0, -0.0),
            (torch.arange(V) % 2048 < 8).float() + (torch.arange(V) // 2048) / 512.0]
    x = torch.stack([r.float() for r in rows]).cuda()
    t = torch.zeros(len(rows), dtype=torch.int64, device="cuda")
    for top in (1, 8, 32):
        out = token_log_probs(x, t, None, 1.0, top)
        check(x, t, None, 1.0, out, top)


@pytest.mark.parametrize("V", [5, 43, 700, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_allowed_tokens(V, dtype):
    """Rows that allow none, one, or fewer than the alternatives asked for; what is masked counts nowhere, infinities and NaN among it."""
    x, t, _, g, h = problem(V, (6,), V, dtype, None)
    mask = torch.zeros(6, V, dtype=torch.bool, device="cuda")
    mask[1, V - 1] = mask[2, 0] = mask[2, V // 2] = mask[3, 1:4] = mask[4] = True
    t = torch.tensor([0, V - 1, 1, 2, V // 2, 0], device="cuda")
    mask[5, 1:] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max], device="cuda")
    x = torch.where(mask, x, bad.to(dtype)[torch.arange(V, device="cuda") % 5])
    want = torch.where(mask, x, 0)
    top = min(V, 8)
    out, grad = run(x, t, mask, 1.0, top, g, h)
    check(want, t, mask, 1.0, out, top, grad, g, h)
    assert out.log_prob[0] == out.log_prob[2] == -float("inf") and out.entropy[0] == out.entropy[1] == 0
    assert float(out.log_prob[1].detach()) == 0 and (out.top_tokens[0] == -1).all()
    # the same from logits of -inf
    same, grad2 = run(torch.where(mask, x, -float("inf")), t, None, 1.0, top, g, h)
    assert all(torch.equal(a, b) for a, b in zip((*out, grad), (*same, grad2)))


@pytest.mark.parametrize("V", [43, 700, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lowest_values_are_values(V, dtype):
    """A mask added as the type's lowest value: one allowed token, and a row of nothing else, which is uniform."""
    low = torch.finfo(dtype).min
    x = torch.full((2, V), low, dtype=dtype, device="cuda")
    x[0, 3] = 1.0
    t = torch.tensor([3, 3], device="cuda")
    g = h = torch.ones(2, device="cuda")
    out, grad = run(x, t, None, 0.5, 2, g, h)
    want = np.log(1 / V)
    np.testing.assert_allclose(np64(out.log_prob), [0, want], atol=1e-6, rtol=1e-6)
    np.testing.assert_allclose(np64(out.entropy), [0, -want], atol=1e-6, rtol=1e-6)
    assert out.top_tokens.tolist() == [[3, 0], [0, 1]] and torch.isfinite(grad).all()


@pytest.mark.parametrize("V", [43, 700, 70000])
def test_a_bad_row_stays_alone(V):
    x, t, m, g, h = problem(1, (9,), V, F32, None)
    t = t.abs()
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[4, 5] = bad
        want, dwant = run(x, t, m, 1.0, 3, g, h)
        out, grad = run(y, t, m, 1.0, 3, g, h)
        assert out.log_prob[4].isnan() and out.entropy[4].isnan() and grad[4].isnan().any()
        keep = torch.arange(9, device="cuda") != 4
        for a, b in zip((*out, grad), (*want, dwant)):
            assert torch.equal(a[keep], b[keep])


def test_peaked_rows():
    """Rows whose probability is all but on one token: no NaN of 0 times a far exponent."""
    for V in (43, 700, 9000):
        x = torch.zeros(3, V, device="cuda")
        x[0, 1], x[1, 1], x[2] = 1e4, 1e38, -1e38
        x[2, 0] = 1e38
        t = torch.tensor([1, 0, 0], device="cuda")
        out, grad = run(x, t, None, 1.0, 2, torch.ones(3, device="cuda"), torch.ones(3, device="cuda"))
        assert out.entropy.abs().max() == 0 and out.log_prob[0] == out.log_prob[2] == 0 and torch.isfinite(grad).all()
        np.testing.assert_allclose(float(out.log_prob[1].detach()), -1e38, rtol=1e-6)


def test_strides_and_cotangents_of_any_layout():
    """Logits without the last step, a step-major batch, columns not side by side, masks of one batch or one column, one used output."""
    gen = torch.Generator().manual_seed(2)
    for V in (43, 1001):
        whole = torch.randn(7, 4, V, generator=gen).cuda()
        t = torch.randint(0, V, (4, 6), generator=gen).cuda()
        masks = [(torch.rand(s, generator=gen) < 0.7).cuda() for s in ((4, 1, V), (1, 6, 1), (V,))]
        for x in (whole.transpose(0, 1)[:, :-1], whole.permute(1, 2, 0).contiguous().transpose(1, 2)[:, 1:]):
            for m in masks:
                g = torch.randn(6, 4, generator=gen).cuda().t()
                out, grad = run(x, t, m, 1.0, 4, g, g[:1].expand(4, 6))
                check(x, t, m, 1.0, out, 4, grad, g, g[:1].expand(4, 6))
        leaf = x.detach().requires_grad_()
        zero = torch.zeros(4, 6, device="cuda")
        for i, cots in ((0, (torch.ones_like(zero), zero)), (1, (zero, torch.ones_like(zero)))):
            got = torch.autograd.grad(token_log_probs(leaf, t)[i].sum(), leaf)[0]
            assert torch.equal(got, torch.autograd.grad(list(token_log_probs(leaf, t)[:2]), leaf, cots)[0])


def test_top_alternatives_have_no_gradient():
    leaf = torch.randn(2, 9, device="cuda").requires_grad_()
    out = token_log_probs(leaf, torch.zeros(2, dtype=torch.int64, device="cuda"), top=2)
    assert out.log_prob.requires_grad and not out.top_log_probs.requires_grad and not out.top_tokens.requires_grad


def test_empty_batches():
    for lead in ((0,), (0, 3), (2, 0)):
        leaf = torch.zeros(*lead, 9, device="cuda").requires_grad_()
        out = token_log_probs(leaf, torch.zeros(lead, dtype=torch.int32, device="cuda"), top=3)
        assert out.top_tokens.shape == (*lead, 3) and out.log_prob.shape == lead
        assert torch.autograd.grad(out.entropy.sum(), leaf)[0].shape == leaf.shape


def test_a_captured_pass_replays():
    for V, top in ((43, 5), (20011, 5), (2000, 0), (70001, 9)):
        sets = [problem(i, (4, 3), V, BF16, "rows") for i in range(3)]
        want = []
        for x, t, m, g, h in sets:
            out, grad = run(x, t, m, 1.0, top, g, h)
            want.append([a.detach().clone() for a in (*out, grad) if a is not None])
            del out, grad
        hold = [a.clone() for a in sets[0]]
        hold[0].requires_grad_()

        def both():
            x, t, m, g, h = hold
            out = token_log_probs(x, t, m, 1.0, top)
            got = (*out, torch.autograd.grad([out.log_prob, out.entropy], x, [g, h])[0])
            return [a for a in got if a is not None]

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
                for a, b in zip(hold, sets[i]):
                    a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def test_on_another_stream():
    x, t, m, g, h = problem(3, (64,), 60000, BF16, "one")
    want = token_log_probs(x, t, m, 1.0, 8)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = token_log_probs(x, t, m, 1.0, 8)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_logits_past_32_bit_offsets():
    """Over 2^31 logits: rows at the end as those of a small batch."""
    V, rows = 65536, 33000
    x = torch.zeros(rows, V, dtype=BF16, device="cuda")
    tail, t, _, g, h = problem(4, (5,), V, BF16, None)
    x[-5:] = tail
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    tokens[-5:] = t
    ones = torch.zeros(rows, device="cuda")
    gg, hh = ones.clone(), ones.clone()
    gg[-5:], hh[-5:] = g, h
    out, grad = run(x, tokens, None, 1.0, 4, gg, hh)
    want, dwant = run(tail, t, None, 1.0, 4, g, h)
    check(tail, t, None, 1.0, want, 4, dwant, g, h)
    assert torch.allclose(out.log_prob[-5:], want.log_prob, rtol=1e-6) and torch.equal(out.top_tokens[-5:], want.top_tokens)
    assert (grad[-5:].float() - dwant.float()).abs().max() <= 2.0 ** -7 * dwant.float().abs().max()

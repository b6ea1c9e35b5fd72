"""token_logprobs (naylis_mom_logprobs_*) against fp64 log-softmax: vocabularies
around the 16-byte chunks and the tiles, strided and unaligned rows, masked
columns, ties, gradients."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (7, 9), (2, 1000), (33, 4097), (16, 32768), (3, 50001), (5, 65536), (2, 151999)]


def _rows(N, V, dtype, dev, seed=0, std=3.0):
    g = torch.Generator(device=dev).manual_seed(seed + V)
    x = torch.randn(N, V, generator=g, device=dev) * std
    x[:, V // 2:] += 2
    return x.to(dtype), torch.randint(0, V, (N,), generator=g, device=dev)


def _reference(x, tok):
    """fp64 log probabilities, entropies, and the bounds of their fp32 errors:
    s sums V / 512 + 80 values of a thread and the joins, each addition and each
    e^d (its exponent d log2 e is rounded once) within 2^-23 of itself; x - m,
    log s and their difference are rounded once each."""
    x = x.double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    m = x.amax(-1)
    d = torch.where(p > 0, p * (x - m[:, None]), 0.0).abs().sum(-1)
    s_err = (x.shape[1] / 512 + 80 + 2 * d) * 2.0 ** -23
    got = lp.gather(1, tok[:, None])[:, 0]
    scale = got.abs() + torch.logsumexp(x - m[:, None], -1).abs()
    return lp, p, got, entropy, s_err + scale * 2.0 ** -22, 2 * s_err * (1 + d) + (scale * 0 + d + 12) * 2.0 ** -22


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_logprobs_match_fp64(N, V, dtype, dev):
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(N, V, dtype, dev)
    if V > 100:
        x[:, 5:V // 50] = -math.inf  # masked columns
        tok = torch.where((tok >= 5) & (tok < V // 50), 0, tok)
    top = min(V, 20)
    r = token_logprobs(x, tok, top=top)
    lp, p, want, entropy, e1, e2 = _reference(x, tok)
    assert bool(((r.logp.double() - want).abs() <= e1).all()), float(((r.logp.double() - want).abs() / e1).max())
    assert bool(((r.entropy.double() - entropy).abs() <= e2).all()), float(((r.entropy.double() - entropy).abs() / e2).max())
    best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(r.top_ids, best)
    bound = e1[:, None] + lp.gather(1, best).abs() * 2.0 ** -21
    assert bool(((r.top_logp.double() - lp.gather(1, best)).abs() <= bound).all())
    again = token_logprobs(x, tok)
    assert again.top_ids is None and again.top_logp is None
    assert torch.equal(again.logp, r.logp) and torch.equal(again.entropy, r.entropy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_logprobs_gradient_matches_fp64(N, V, dtype, dev):
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(N, V, dtype, dev, seed=1)
    if V > 100:
        x[:, 5:V // 50] = -math.inf
        tok = torch.where((tok >= 5) & (tok < V // 50), 0, tok)
    g = torch.Generator(device=dev).manual_seed(2)
    gl, ge = (torch.randn(N, generator=g, device=dev) for _ in range(2))
    x.requires_grad_()
    r = token_logprobs(x, tok)
    both, = torch.autograd.grad((r.logp, r.entropy), x, (gl, ge), retain_graph=True)
    one, = torch.autograd.grad(r.logp, x, gl, retain_graph=True)
    other, = torch.autograd.grad(r.entropy, x, ge)
    lp, p, _, entropy, e1, e2 = _reference(x.detach(), tok)
    hot = torch.zeros_like(lp).scatter_(1, tok[:, None], 1.0)
    plp = torch.where(p > 0, p * (lp + entropy[:, None]), 0.0)
    pa = torch.where(p > 0, p * (lp.abs() + entropy[:, None] + 1), 0.0)
    half = torch.finfo(dtype).eps / 2
    for got, a, b in ((both, gl, ge), (one, gl, 0 * ge), (other, 0 * gl, ge)):
        a, b = a.double()[:, None], b.double()[:, None]
        want = a * (hot - p) - b * plp
        # the result's rounding; p's relative error, that of its exponent (e1 + e2 of lp + H)
        err = half * want.abs() + (e1 + e2 + 2.0 ** -20)[:, None] * (a.abs() * (hot + p) + b.abs() * pa) + 1e-44
        assert bool(((got.double() - want).abs() <= err).all()), float(((got.double() - want).abs() / err).max())


def test_logprobs_gradient_matches_differences(dev):
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(6, 777, torch.float32, dev, seed=4)
    g = torch.Generator(device=dev).manual_seed(5)
    gl, ge = (torch.randn(6, generator=g, device=dev) for _ in range(2))
    u = torch.randn(6, 777, generator=g, device=dev, dtype=torch.float64)

    def value(y):
        lp = torch.log_softmax(y, -1)
        return float((lp.gather(1, tok[:, None])[:, 0] * gl).sum() - ((lp.exp() * lp).sum(-1) * ge).sum())

    slope = (value(x.double() + 1e-5 * u) - value(x.double() - 1e-5 * u)) / 2e-5
    x.requires_grad_()
    r = token_logprobs(x, tok)
    d, = torch.autograd.grad((r.logp, r.entropy), x, (gl, ge))
    # fp32 gradient: at most 2^-16 of the terms' magnitudes (the bound above), terms under 40
    assert abs(float((d.double() * u).sum()) - slope) < 40 * float(u.abs().sum(-1).max()) * 2.0 ** -16


@pytest.mark.parametrize("V", [5003, 70001])  # rows in one piece, and cut into parts
def test_logprobs_ties_masks_and_nan(V, dev):
    """Equal logits (more than the ranking holds at once), rows of -inf, NaN,
    infinities, signed zeros: the order of a stable descending sort."""
    from naylis_amd.mom_kernels import token_logprobs
    g = torch.Generator(device=dev).manual_seed(0)
    rows = torch.zeros(9, V, device=dev)
    rows[1] = torch.randint(0, 3, (V,), generator=g, device=dev)
    rows[2, ::2] = -0.0
    rows[3] = -math.inf
    rows[3, 4000:4010] = 1.0
    rows[4] = -math.inf
    rows[5] = torch.arange(V, device=dev) // 500
    rows[6] = torch.randn(V, generator=g, device=dev)
    rows[6, [7, 4999]] = math.nan
    rows[7] = torch.randn(V, generator=g, device=dev)
    rows[7, 100] = math.inf
    rows[8] = torch.randn(V, generator=g, device=dev)
    tok = torch.full((9,), 4001, device=dev)
    for dtype in (torch.bfloat16, torch.float32):
        for top in (1, 17, 64):
            x = rows.to(dtype)
            r = token_logprobs(x, tok, top=top)
            best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
            assert torch.equal(r.top_ids, best)
            assert bool(r.logp[[4, 6, 7]].isnan().all() and r.entropy[[4, 6, 7]].isnan().all())
            assert bool(r.logp[[0, 1, 2, 3, 5, 8]].isfinite().all())
            # ten equal logits among -inf: log 10, and -inf for the others
            assert abs(float(r.logp[3]) + math.log(10)) < 1e-6 and abs(float(r.entropy[3]) - math.log(10)) < 1e-6
            assert top <= 10 or bool((r.top_logp[3, 10:] == -math.inf).all())
            assert abs(float(r.entropy[0]) - math.log(V)) < 1e-4  # V / 512 additions and more, each 2^-24


@pytest.mark.parametrize("V", [70, 5003, 70001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logprobs_nan_in_the_first_column(dtype, V, dev):
    """A NaN in column 0 comes first like any other: rows of NaN, of -inf with a
    NaN, of equal logits with a NaN (more of them than the ranking holds at once)."""
    from naylis_amd.mom_kernels import token_logprobs
    x = torch.full((5, V), math.nan, dtype=dtype, device=dev)
    x[1] = -math.inf
    x[2] = 1.0
    x[1:3, 0] = math.nan
    x[3] = -math.inf
    x[3, [0, 60, V - 1]] = math.nan
    x[4, V // 2:] = 0.0
    for top in (1, 17, 64):
        got = token_logprobs(x, torch.zeros(5, dtype=torch.long, device=dev), top=top)
        assert torch.equal(got.top_ids, torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]), top
        assert bool(got.logp.isnan().all() and got.entropy.isnan().all() and got.top_logp.isnan().all())


@pytest.mark.parametrize("V", [1003, 70001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logprobs_of_lowest_values(dtype, V, dev):
    """Masks of the type's lowest value: nothing beside other logits, an even row
    by themselves; large logits either way; gradients finite."""
    from naylis_amd.mom_kernels import token_logprobs
    low = torch.finfo(dtype).min
    x = torch.full((5, V), low, dtype=dtype, device=dev)
    x[1, 10:20] = 1.0
    x[2] = -low
    x[3] = -1e4
    x[3, 5] = 1e4
    x[4, ::2] = -math.inf
    tok = torch.tensor([7, 12, V - 1, 5, 1], device=dev)
    x.requires_grad_()
    r = token_logprobs(x, tok, top=3)
    want = [-math.log(V), -math.log(10), -math.log(V), 0.0, -math.log(V // 2)]
    for i, w in enumerate(want):  # V / 512 + 80 fp32 additions in the sum, and log's own steps
        bound = (V / 512 + 80) * 2.0 ** -23 + 12 * 2.0 ** -22
        assert abs(float(r.logp[i].detach()) - w) < bound and abs(float(r.entropy[i].detach()) + w) < bound, i
    assert r.top_ids.tolist() == [[0, 1, 2], [10, 11, 12], [0, 1, 2], [5, 0, 1], [1, 3, 5]]
    d, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x)
    assert bool(d.isfinite().all()) and bool((d[1, 20:] == 0).all()) and bool((d[4, ::2] == 0).all())
    assert abs(float(d[0, 7]) - (1 - 1 / V)) < 2.0 ** -8


@pytest.mark.parametrize("V", [9, 1003, 70001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logprobs_of_logits_of_any_size(dtype, V, dev):
    """Logits past 2^24, where x log2 e is off by more than 1: rows of a few far
    values apart, close together, on both sides of 2^24, up to the type's ends, and
    tokens masked by a large negative number; against fp64 of the same values.

    Bounds: of e^(x - m), x - m is exact where it matters (fp32, under 2^7, and its
    operands within a factor of two), so the sums' errors are those of _reference; a
    log probability of -d with d large is one rounding of x - m, one of it less log
    s and two of a product with log2 e and back (2^-22 d in all); of the near rows,
    whose reference is rounded, d itself is off by 2^-24 of the logits' size."""
    from naylis_amd.mom_kernels import token_logprobs
    low, big = torch.finfo(dtype).min, torch.finfo(dtype).max
    step = 2.0 ** 24 * torch.finfo(dtype).eps  # neighbouring values at 2^24
    rows = [[2e7, 3e7], [-3e7, -2e7], [2.0 ** 24, 2.0 ** 24 + 2 * step], [2.0 ** 24, 2.0 ** 24 - step],
            [-2.0 ** 24 - 2 * step, -2.0 ** 24 + step], [1e30, 1.5e30], [low, 0.0], [low, 5.0], [-1e9, 3.0],
            [low, big], [big, big], [low, low], [-1e30, 2e7], [-2e7, 1e7], [0.0, 1e38]]
    g = torch.Generator(device=dev).manual_seed(9)
    pick = torch.randint(0, 2, (len(rows), V), generator=g, device=dev)
    pick[:, 0], pick[:, 1], pick[:, V - 1] = 0, 1, 0
    x = torch.tensor(rows, dtype=torch.float64, device=dev).to(dtype).gather(1, pick)
    x[:, 3] = -math.inf
    x.requires_grad_()
    z = x.detach().double()
    for col in (0, 1, V - 1):
        tok = torch.full((len(rows),), col, device=dev)
        r = token_logprobs(x, tok, top=5)
        lp = torch.log_softmax(z, -1)
        p = lp.exp()
        want, entropy = lp[:, col], -torch.where(p > 0, p * lp, 0.0).sum(-1)
        m = z.amax(-1)
        near = torch.where(m.abs() <= 2.0 ** 24, m.abs(), 0.0) * 2.0 ** -22
        d = torch.where(p > 0, p * (z - m[:, None]), 0.0).abs().sum(-1)
        s_err = (V / 512 + 80 + 2 * d) * 2.0 ** -23
        err = s_err + want.abs() * 2.0 ** -22 + math.log(V) * 2.0 ** -22 + torch.where(want < -1, near, 0.0)
        fits = want.float().isfinite()  # (low less big rounds to no fp32 number; low less a logarithm rounds to low)
        assert bool((r.logp.double() - want).abs()[fits].le(err[fits]).all()), (r.logp, want)
        assert bool((r.logp[~fits] == -math.inf).all())
        assert bool(((r.entropy.double() - entropy).abs() <= 2 * s_err * (1 + d) + (d + 12) * 2.0 ** -22).all())
        assert torch.equal(r.top_ids, torch.sort(x.detach(), dim=-1, descending=True, stable=True)[1][:, :5])
        dx, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x)
        hot = torch.zeros_like(lp)
        hot[:, col] = 1
        grad = hot - p - torch.where(p > 0, p * (lp + entropy[:, None]), 0.0)
        size = hot + p + torch.where(p > 0, p * (lp.abs() + entropy[:, None]), 0.0)
        tol = torch.finfo(dtype).eps / 2 * grad.abs() + (s_err * (3 + d) + (d + 12) * 2.0 ** -21)[:, None] * size + 1e-30
        assert bool(((dx.double() - grad).abs() <= tol).all()), float(((dx.double() - grad).abs() / tol).max())


def test_logprobs_ignored_and_bad_tokens(dev):
    from naylis_amd.mom_kernels import token_logprobs
    x, _ = _rows(5, 300, torch.bfloat16, dev)
    tok = torch.tensor([3, -100, 300, -1, 299], device=dev)
    x.requires_grad_()
    r = token_logprobs(x, tok)
    assert float(r.logp[1].detach()) == 0 and bool(r.logp[2:4].isnan().all()) and bool(r.entropy.isfinite().all())
    d, = torch.autograd.grad(r.logp, x, torch.ones(5, device=dev), retain_graph=True)
    assert bool((d[1] == 0).all() and d[2:4].isnan().all() and d[[0, 4]].isfinite().all())
    d, = torch.autograd.grad(r.entropy, x, torch.ones(5, device=dev))
    assert bool(d[1].abs().sum() > 0)
    r = token_logprobs(x, tok, ignore_index=299)
    assert float(r.logp[4].detach()) == 0 and bool(r.logp[1:4].isnan().all())
    d, = torch.autograd.grad(r.logp[4], x)  # bad tokens' rows are NaN for any incoming gradient
    assert bool((d[[0, 4]] == 0).all() and d[1:4].isnan().all())


@pytest.mark.parametrize("V", [7, 300, 70001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logprobs_ignored_rows_without_probabilities(dtype, V, dev):
    """Padding rows of -inf or NaN, or with an infinity, whose token is ignored:
    log probability 0, and a gradient of exactly 0 from it."""
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(6, V, dtype, dev)
    x[1] = -math.inf
    x[2, V // 2] = math.nan
    x[3] = math.nan
    x[4, 3] = math.inf
    tok[1:5] = -100
    wide = torch.zeros(6, V + 3, dtype=dtype, device=dev)
    wide[:, 1:V + 1] = x
    for y in (x, wide[:, 1:V + 1].detach()):  # rows at the gradient's alignment, and at others
        y.requires_grad_()
        r = token_logprobs(y, tok)
        assert bool((r.logp[1:5] == 0).all() and r.entropy[1:5].isnan().all())
        d, = torch.autograd.grad(r.logp, y, torch.ones(6, device=dev), retain_graph=True)
        assert bool((d[1:5] == 0).all() and d.isfinite().all() and d[[0, 5]].any(-1).all())
        some = torch.tensor([1.0, 0.0, 0.0, 0.0, 0.0, 0.5], device=dev)  # the ignored rows' entropies are left out
        d, = torch.autograd.grad((r.logp, r.entropy), y, (torch.ones(6, device=dev), some))
        assert bool((d[1:5] == 0).all() and d.isfinite().all() and d[[0, 5]].any(-1).all())


def test_logprobs_views_and_shapes(dev):
    """Rows of a padded buffer (any stride and address), leading dimensions,
    int32 tokens, sums' expanded gradients, streams."""
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(6, 1001, torch.bfloat16, dev)
    want = token_logprobs(x, tok, top=5)
    wide = torch.zeros(6, 1030, dtype=torch.bfloat16, device=dev)
    for off in range(1, 9):
        wide[:, off:off + 1001] = x
        y = wide[:, off:off + 1001].detach().requires_grad_()
        got = token_logprobs(y, tok.int(), top=5)
        # sums over chunks cut elsewhere: the fp32 bounds of both sides
        e1, e2 = _reference(x, tok)[4:]
        assert bool(((got.logp - want.logp).abs() <= 2 * e1).all()) and torch.equal(got.top_ids, want.top_ids)
        assert bool(((got.entropy - want.entropy).abs() <= 2 * e2).all())
        d, = torch.autograd.grad((got.logp.sum() + got.entropy.sum()), y)
        z = x.clone().requires_grad_()
        r = token_logprobs(z, tok)
        dz, = torch.autograd.grad((r.logp, r.entropy), z, (torch.ones(6, device=dev), torch.ones(6, device=dev)))
        assert float((d.float() - dz.float()).norm() / dz.float().norm()) < 2.0 ** -8
    wide32 = torch.zeros(6, 1010, device=dev)
    wide32[:, 3:1004] = x.float()
    assert torch.equal(token_logprobs(wide32[:, 3:1004], tok, top=5).top_ids, want.top_ids)
    lead = token_logprobs(x.view(2, 3, 1001), tok.view(2, 3), top=5)
    assert lead.logp.shape == (2, 3) and lead.top_ids.shape == (2, 3, 5) and torch.equal(lead.logp.flatten(), want.logp)
    flat = token_logprobs(x[0], tok[0], top=5)
    assert flat.logp.shape == () and torch.equal(flat.top_ids, want.top_ids[0])
    t = x.t().contiguous().t()  # columns not dense: copied
    assert torch.equal(token_logprobs(t, tok).logp, want.logp)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = token_logprobs(x, tok, top=5)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    e = token_logprobs(x[:0], tok[:0], top=5)
    assert e.logp.shape == (0,) and e.top_ids.shape == (0, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logprobs_far_rows(dtype, dev):
    """Rows further than 2^31 elements and 2^32 bytes from the first."""
    from naylis_amd.mom_kernels import token_logprobs
    N, V, ld = 300, 1000, (1 << 23) - 5
    x = torch.randn(N, V, generator=torch.Generator(device=dev).manual_seed(2), device=dev).to(dtype)
    far = torch.as_strided(torch.empty(N * ld, dtype=dtype, device=dev), (N, V), (ld, 1)).copy_(x)
    tok = torch.arange(N, device=dev)
    y, z = x.requires_grad_(), far.requires_grad_()
    a, b = token_logprobs(y, tok, top=5), token_logprobs(z, tok, top=5)
    assert torch.equal(a.top_ids, b.top_ids)
    for s, t in ((a.logp, b.logp), (a.entropy, b.entropy), (a.top_logp, b.top_logp)):
        # the same values on other chunks: the sums' order differs (at most V / 256 + 16 additions)
        assert float((s - t).detach().abs().max()) <= 2 * ((V / 256 + 16) * 2.0 ** -23 + 12 * 2.0 ** -22)
    ga, = torch.autograd.grad(a.logp.sum(), y)
    gb, = torch.autograd.grad(b.logp.sum(), z)
    assert float((ga.float() - gb.float()).abs().max()) <= torch.finfo(dtype).eps + 2.0 ** -18


def test_logprobs_graph(dev):
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(8, 4099, torch.bfloat16, dev)
    held, ht = x.clone().requires_grad_(), tok.clone()
    gl, ge = torch.ones(8, device=dev), torch.ones(8, device=dev)

    def run(a, t):
        r = token_logprobs(a, t, top=10)
        d, = torch.autograd.grad((r.logp, r.entropy), a, (gl, ge))
        return [r.logp.detach(), r.entropy.detach(), r.top_ids, r.top_logp, d]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(held, ht)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs = run(held, ht)
    for seed in range(4):
        y, t = _rows(8, 4099, torch.bfloat16, dev, seed=10 * seed, std=0.01 if seed == 2 else 3.0)
        with torch.no_grad():
            held.copy_(y)
        ht.copy_(t)
        eager = run(y.requires_grad_(), t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), seed


def test_logprobs_agree_with_the_loss(dev):
    """cross_entropy_rows of the same rows, within both kernels' fp32 bounds."""
    from naylis_amd.mom_kernels import token_logprobs
    from naylis_amd.mom_kernels.hip_xent import cross_entropy_rows
    x, tok = _rows(9, 4096, torch.bfloat16, dev)
    e1 = _reference(x, tok)[4]
    assert bool(((token_logprobs(x, tok).logp + cross_entropy_rows(x, tok)).abs() <= 2 * e1 + 2.0 ** -19).all())


def test_logprobs_refusals(dev):
    from naylis_amd.mom_kernels import token_logprobs
    x, tok = _rows(4, 100, torch.bfloat16, dev)
    for args, kw in (((x.half(), tok), {}), ((x, tok[:3]), {}), ((x, tok.cpu()), {}), ((x, tok.float()), {}),
                     ((x[:, :0], tok), {}), ((x, tok), {"top": 101}), ((x, tok), {"top": -1}), ((x, tok), {"top": 65})):
        with pytest.raises(RuntimeError, match="logprobs"):
            token_logprobs(*args, **kw)
    x.requires_grad_()
    r = token_logprobs(x, tok)
    g, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(g.float().sum(), x)

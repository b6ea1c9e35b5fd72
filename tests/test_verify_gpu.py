"""verify_drafts against a statement of the rule in fp64, one sequence at a time:
drafts of a model and of a rule, greedy rows, odd vocabularies and addresses,
rows without a distribution; and that the tokens come out as the model's own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(B, N, V, dtype, probs, dev, seed=0, std=2.0):
    g = torch.Generator(device=dev).manual_seed(seed + 1000 * B + N + V)
    x = torch.randn(B, N + 1, V, generator=g, device=dev) * std
    hot = torch.randint(0, V, (B, N + 1, min(8, V)), generator=g, device=dev)
    x.scatter_add_(2, hot, 4 + 6 * torch.rand(hot.shape, generator=g, device=dev))
    q = None
    if probs is not None:
        q = torch.softmax(x[:, :N] + torch.randn(B, N, V, generator=g, device=dev) * 0.7, -1).to(probs)
    x = x.to(dtype)
    best = x[:, :N].float().argmax(-1) if N else torch.zeros(B, 0, dtype=torch.long, device=dev)
    drafts = torch.where(torch.rand(B, N, generator=g, device=dev) < 0.7, best, hot[:, :N, 0])
    return dict(logits=x, drafts=drafts, uniforms=torch.rand(B, N + 1, generator=g, device=dev), draft_probs=q)


def _rule(c, B, draft_lens=None, temperature=1.0):
    """The rule in fp64 for each sequence: (tokens, accepted, how near the random
    numbers come to a border that would change them, relative to the whole)."""
    x, d, u, q = (c[n] if c[n] is None else c[n].cpu() for n in ("logits", "drafts", "uniforms", "draft_probs"))
    N = d.shape[1]
    tokens, accepted, margin = torch.full((B, N + 1), -1), torch.zeros(B, dtype=torch.int32), torch.full((B,), math.inf)
    for b in range(B):
        n = N if draft_lens is None else min(max(int(draft_lens[b]), 0), N)
        t = float(torch.as_tensor(temperature, dtype=torch.float32).expand(B)[b])

        def dist(i):
            row = x[b, i].double()
            if row.isnan().any() or row.max() == math.inf or row.max() == -math.inf:
                return None
            if t > 0:
                return torch.softmax((row - row.max()) / t, 0)
            p = torch.zeros_like(row)
            p[int((row == row.max()).nonzero()[0])] = 1
            return p
        a, w = 0, None
        while a < n:
            p, i = dist(a), int(d[b, a])
            if p is None:
                break
            w = None
            if 0 <= i < len(p):
                ratio = float(u[b, a]) * (1.0 if q is None else float(q[b, a, i]))
                margin[b] = min(margin[b], abs(ratio - float(p[i])))
                if ratio < float(p[i]):
                    a += 1
                    continue
            if q is not None:
                w = (p - q[b, a].double()).clamp(min=0)
            else:
                w = p.clone()
                if 0 <= i < len(p):
                    w[i] = 0
            break
        p = dist(a)
        accepted[b] = a
        tokens[b, :a] = d[b, :a]
        if p is None:
            continue
        if a == n or w is None or float(w.sum()) == 0:
            w = p
        cum = torch.cumsum(w, 0)
        target = float(u[b, N]) * float(cum[-1])
        at = int(torch.searchsorted(cum, torch.tensor(target, dtype=torch.float64), right=True))
        tokens[b, a] = min(at, int(w.nonzero()[-1]))
        if t > 0:
            margin[b] = min(margin[b], float((cum - target).abs().min()) / max(float(cum[-1]), 1e-300))
    return tokens, accepted, margin


def _check(c, dev, **kw):
    from naylis_amd.mom_kernels import verify_drafts
    B = len(c["drafts"])
    got = verify_drafts(c["logits"], c["drafts"], c["uniforms"], draft_probs=c["draft_probs"], **kw)
    want, accepted, margin = _rule(c, B, **{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    # both sides sum up to 2^18 weights in fp64, each off by less than 2^-50 of itself:
    # a border is off by less than 2^-40 of the whole.  p - q may be far smaller than
    # both: its own whole is at least the 2^-20 or so that a rejection leaves here
    clear = margin > 2.0 ** -38
    assert int((~clear).sum()) <= B // 50, "the inputs put random numbers next to borders"
    assert got.tokens.dtype == torch.int64 and got.accepted.dtype == torch.int32
    assert torch.equal(got.tokens.cpu()[clear], want[clear]), (got.tokens.cpu()[clear] != want[clear]).any(-1).nonzero()
    assert torch.equal(got.accepted.cpu()[clear], accepted[clear])
    again = verify_drafts(c["logits"], c["drafts"], c["uniforms"], draft_probs=c["draft_probs"], **kw)
    assert torch.equal(got.tokens, again.tokens) and torch.equal(got.accepted, again.accepted)
    return got


SHAPES = [(1, 0, 1), (1, 1, 2), (3, 2, 7), (5, 3, 8), (2, 8, 1000), (70, 4, 2047), (3, 1, 2048), (3, 2, 2049), (2, 3, 4096),
          (9, 5, 8191), (4, 2, 50001), (2, 1, 151999), (1, 12, 32768), (2, 40, 513), (3, 95, 500), (2, 100, 9001), (5, 0, 24000),
          (5, 0, 24700), (4, 3, 12281), (4, 3, 12282), (5, 0, 8185), (5, 0, 8186), (4, 3, 4089), (4, 3, 4090), (4, 3, 9209),
          (4, 3, 9210), (3, 47, 500), (3, 48, 500), (2, 109, 500), (2, 110, 500),
          (5, 0, 10233), (5, 0, 10234), (5, 1, 7673), (5, 1, 7674)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16], ids=["rule", "q32", "q16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_verify_matches_the_rule(shape, probs, dtype, dev):
    _check(_case(*shape, dtype, probs, dev), dev)


@pytest.mark.parametrize("probs", [None, torch.float32], ids=["rule", "q32"])
def test_verify_wide_batches(probs, dev):
    """Enough rows for the larger parts of a row, with lengths, temperatures and
    greedy sequences of their own."""
    B, N, V = 40, 5, 40000
    c = _case(B, N, V, torch.bfloat16, probs, dev)
    t = torch.rand(B, device=dev, generator=torch.Generator(device=dev).manual_seed(3)) + 0.3
    t[::5] = 0
    lens = torch.tensor([(i % 8) - 1 for i in range(B)], dtype=torch.int32, device=dev)
    got = _check(c, dev, draft_lens=lens, temperature=t)
    assert bool((got.accepted <= lens.clamp(0, N)).all()) and int(got.accepted.max()) > 1
    _check(c, dev, draft_lens=lens.long(), temperature=0.7)


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 3.0, 100.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_verify_temperatures(dtype, temperature, dev):
    _check(_case(20, 3, 3001, dtype, torch.float32, dev), dev, temperature=temperature)


@pytest.mark.parametrize("probs", [None, torch.float32], ids=["rule", "q32"])
@pytest.mark.parametrize("B,V", [(4, 3001), (4, 50001), (150, 33001)])  # one launch; in two or three; in three
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_verify_temperatures_at_the_ends(dtype, B, V, probs, dev):
    """The least that fp32 holds takes the largest logit, infinity all columns alike."""
    c = _case(B, 3, V, dtype, probs, dev)
    c["logits"][..., 77] = 60.0  # the one largest
    ends = torch.tensor([2.0 ** -149, 2.0 ** -130, 3e38, math.inf], device=dev)
    _check(c, dev, temperature=ends[torch.arange(B, device=dev) % 4])


@pytest.mark.parametrize("probs", [None, torch.float32], ids=["rule", "q32"])
@pytest.mark.parametrize("B,V", [(4, 3001), (4, 50001), (150, 33001)])  # one launch; in two or three; in three
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_verify_temperatures_of_any_size(dtype, B, V, probs, dev):
    """Logits up to the largest numbers and down to the smallest with temperatures of their
    size: differences beyond fp32's largest number, scales beyond it."""
    g = torch.Generator(device=dev).manual_seed(V)
    for size, t in ((2.0 ** 127, 2.0 ** 126), (2.0 ** 127, 2.0 ** 127 * 1.9), (2.0 ** 127, math.inf), (2.0 ** 110, 2.0 ** 109),
                    (2.0 ** -95, 2.0 ** -96), (2.0 ** -110, 2.0 ** -111), (2.0 ** -125, 2.0 ** -126)):
        x = ((torch.rand(B, 4, V, generator=g, device=dev, dtype=torch.float64) * 2 - 1) * size).to(dtype)
        drafts = x[:, :3].float().argmax(-1)
        drafts[::2] = torch.randint(0, V, drafts[::2].shape, generator=g, device=dev)
        u = torch.rand(B, 4, generator=g, device=dev)
        u[:, :3] /= V  # near the probabilities of a row that is nearly flat
        q = None
        if probs is not None:
            q = torch.rand(B, 3, V, generator=g, device=dev)
            u[:, :3] *= V
            q /= q.sum(-1, keepdim=True)
        got = _check(dict(logits=x, drafts=drafts, uniforms=u, draft_probs=q), dev, temperature=torch.full((B,), t, device=dev))
        # (at infinity every p is 1 / V, and every u / V below it)
        all_kept = t == math.inf and probs is None
        assert B < 150 or (int(got.accepted.sum()) == 3 * B if all_kept else 0 < int(got.accepted.sum()) < 3 * B)


def test_verify_greedy(dev):
    """Temperature 0: drafts are kept while they are the first largest logit, and
    that one follows, with and without probabilities of the drafts."""
    from naylis_amd.mom_kernels import verify_drafts
    g = torch.Generator(device=dev).manual_seed(5)
    B, N, V = 33, 4, 5003
    x = torch.randint(0, 40, (B, N + 1, V), generator=g, device=dev).bfloat16()  # ties in every row
    best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device=dev), V).amin(-1)
    drafts = torch.where(torch.rand(B, N, generator=g, device=dev) < 0.8, best[:, :N], torch.randint(0, V, (B, N), generator=g, device=dev))
    same = (drafts == best[:, :N]).long().cumprod(-1).sum(-1)
    u = torch.rand(B, N + 1, generator=g, device=dev)
    for probs in (None, torch.softmax(x[:, :N].float(), -1), torch.full((B, N, V), 0.99, device=dev)):
        for t in (0, torch.zeros(B, device=dev)):
            r = verify_drafts(x, drafts.int(), u, draft_probs=probs, temperature=t)
            assert torch.equal(r.accepted.long(), same)
            i = torch.arange(N + 1, device=dev)
            assert torch.equal(r.tokens, torch.where(i <= same[:, None], best, -1))


# the first of drafts of a rule, or with probabilities; whether its decision's sums are fp64
DECISIONS = [(40, 1, 7000, False, True), (20, 3, 50001, False, True),
             (40, 3, 2000, False, False), (40, 2, 3000, True, False), (40, 3, 50001, True, False), (150, 3, 33001, False, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,N,V,probs,exact", DECISIONS)
def test_verify_decisions_next_to_their_border(B, N, V, probs, exact, dtype, dev):
    """Random numbers beside p / q: the neighbouring fp32 number on either side where the
    sums are fp64, 2^-18 away where they are fp32 (off by less than 2^-19)."""
    from naylis_amd.mom_kernels import verify_drafts
    c = _case(B, N, V, dtype, torch.float32 if probs else None, dev)
    T, row = 0.83, torch.arange(B, device=dev)
    x, d, q = c["logits"], c["drafts"], c["draft_probs"]
    d[::3, 0] = torch.randint(0, V, (len(d[::3]),), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    t = torch.full((B,), T, device=dev)
    # (on the CPU: on this GPU torch's fp64 softmax is off by up to 1e-6)
    p = torch.softmax(x[:, 0].cpu().double() / t.cpu().double()[:, None], -1).to(dev)[row, d[:, 0]]
    if probs:
        q[row, 0, d[:, 0]] = (1.5 * p).float()
        p = p / q[row, 0, d[:, 0]].double()
    for kept in (True, False):
        if exact:
            u = p.float()
            off = u.double() >= p if kept else u.double() < p  # on the wrong side of p
            u = torch.where(off, torch.nextafter(u, torch.tensor(0.0 if kept else 2.0, device=dev)), u)
        else:
            u = (p * (1 + (-1 if kept else 1) * 2.0 ** -18)).float()
        c["uniforms"][:, 0] = u
        got = verify_drafts(x, d, c["uniforms"], draft_probs=q, temperature=t)
        assert torch.equal(got.accepted > 0, torch.full((B,), kept, device=dev))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_verify_masked_columns(dtype, dev):
    """Columns of -inf are never drawn, the type's lowest value is an ordinary
    logit, and a draft on a masked column is turned away."""
    from naylis_amd.mom_kernels import verify_drafts
    c = _case(64, 3, 2500, dtype, None, dev)
    allowed = torch.zeros(2500, dtype=torch.bool, device=dev)
    allowed[[3, 700, 2047, 2048, 2499]] = True
    for low in (-math.inf, torch.finfo(dtype).min):
        c["logits"] = torch.where(allowed, c["logits"], torch.tensor(low, dtype=dtype, device=dev))
        got = _check(c, dev)
        drawn = got.tokens.gather(1, got.accepted[:, None].long())
        assert bool(allowed[drawn].all()) and bool(allowed[got.tokens[got.tokens >= 0]].all())
    c["logits"] = torch.full_like(c["logits"], torch.finfo(dtype).min)  # all equal, however low
    got = verify_drafts(c["logits"], c["drafts"], c["uniforms"])
    want = (c["uniforms"][:, -1].double() * 2500).floor().long()
    at = got.tokens.gather(1, got.accepted[:, None].long())[:, 0]
    assert int((at - want).abs().max()) <= 1  # (the turned-away draft moves the later ones by one)


@pytest.mark.parametrize("bad", ["nan", "inf", "masked"])
@pytest.mark.parametrize("probs", [None, torch.float32], ids=["rule", "q32"])
@pytest.mark.parametrize("t", [1.0, 0.0])
def test_verify_rows_without_a_distribution(t, probs, bad, dev):
    """Such a row keeps no draft and gives -1; other sequences are untouched."""
    from naylis_amd.mom_kernels import verify_drafts
    V = 3000
    c = _case(6, 2, V, torch.bfloat16, probs, dev)
    x = c["logits"]
    for b, i in ((1, 0), (2, 1), (3, 2)):
        if bad == "masked":
            x[b, i] = -math.inf
        else:
            x[b, i, 2500 if b == 1 else 0] = float(bad)
    c["drafts"][1:4] = x[1:4, :2].float().nan_to_num(0, 0).argmax(-1)
    c["drafts"][2, 1] = 0  # the first of nothing but -inf is no draft to keep
    c["uniforms"][1:4, :2] = 0.0  # anything with a probability is kept
    got = verify_drafts(x, c["drafts"], c["uniforms"], draft_probs=c["draft_probs"], temperature=t)
    assert got.accepted[1:4].tolist() == [0, 1, 2]
    assert got.tokens[1].tolist() == [-1, -1, -1] and got.tokens[2, 1:].tolist() == [-1, -1] and int(got.tokens[3, 2]) == -1
    x[1:4] = 0
    fine = verify_drafts(x, c["drafts"], c["uniforms"], draft_probs=c["draft_probs"], temperature=t)
    for b in (0, 4, 5):
        assert torch.equal(got.tokens[b], fine.tokens[b])


@pytest.mark.parametrize("B,V", [(2, 6100), (2, 10000), (2, 40000), (600, 20000)])  # one launch, sums in fp64, and in fp32
def test_verify_signalling_nans(B, V, dev):
    """NaNs of every bit pattern, one and a whole part of them."""
    from naylis_amd.mom_kernels import verify_drafts
    x = torch.zeros(B, 2, V, dtype=torch.bfloat16, device=dev)
    drafts, u = torch.full((B, 1), 17, device=dev), torch.zeros(B, 2, device=dev)
    for bits in (0x7f81, 0x7fc0, 0xff81 - 65536, 0xffff - 65536):
        for where in (slice(17, 18), slice(V - 1000, V - 999), slice(2048, 6144), slice(None)):
            y = x.clone()
            y.view(torch.int16)[1, 0, where] = bits
            got = verify_drafts(y, drafts, u)
            assert got.accepted[:2].tolist() == [1, 0] and got.tokens[:2].tolist() == [[17, 0], [-1, -1]]


def test_verify_drafts_that_are_none(dev):
    """Ids outside the vocabulary are turned away and take nothing from p."""
    c = _case(40, 3, 900, torch.float32, None, dev)
    c["drafts"][::3, 1] = -1
    c["drafts"][1::3, 0] = 900
    c["drafts"][2::3, 2] = 1 << 40
    got = _check(c, dev)
    assert int(got.accepted[1::3].max()) == 0
    c["draft_probs"] = torch.softmax(c["logits"][:, :3] * 0.5, -1)
    _check(c, dev)


def test_verify_rest_of_nothing(dev):
    """Drafts' probabilities at or above p everywhere: what is left of p is nothing,
    and the token comes from p."""
    c = _case(30, 2, 600, torch.float32, None, dev)
    c["draft_probs"] = torch.full((30, 2, 600), 2.0, device=dev)
    c["uniforms"][:, :2] = 0.999
    got = _check(c, dev)
    assert int(got.accepted.max()) == 0


def test_verify_random_numbers_at_the_ends(dev):
    """0 keeps every draft that has a probability and draws the first column that
    has one; the largest below 1, and 1 itself, draw no column behind the last."""
    from naylis_amd.mom_kernels import verify_drafts
    V = 2100
    x = torch.zeros(2, 2, V, device=dev)
    x[:, :, :5] = x[:, :, V - 3:] = -math.inf
    drafts = torch.tensor([[7], [2]], device=dev)
    u = torch.zeros(2, 2, device=dev)
    assert verify_drafts(x, drafts, u).tokens.tolist() == [[7, 5], [5, -1]]
    for last in (1 - 2.0 ** -24, 1.0):
        u[:, 1] = last
        assert verify_drafts(x, drafts, u).tokens.tolist() == [[7, V - 4], [V - 4, -1]]


@pytest.mark.parametrize("probs", [False, True], ids=["rule", "q32"])
@pytest.mark.parametrize("B,V", [(2, 6100), (2, 12000), (2, 50001), (130, 66001)])  # one launch, two and three
def test_verify_parts_of_next_to_nothing(B, V, probs, dev):
    """A random number of 0 takes the first column with a weight, where the weights of
    many columns together pass what counts as one and each by itself does not."""
    from naylis_amd.mom_kernels import verify_drafts
    x = torch.zeros(B, 2, V, device=dev)
    x[..., :4096] = -905 * math.log(2)  # a weight of 2^-905, of 512 of them 2^-896
    drafts, u = torch.full((B, 1), V - 1, device=dev), torch.zeros(B, 2, device=dev)
    got = verify_drafts(x, drafts, u, draft_probs=torch.full((B, 1, V), 1 / V, device=dev) if probs else None)
    assert got.accepted.tolist() == [1] * B and got.tokens[:, 1].tolist() == [0] * B
    x[..., :4096] = -2000.0  # no weight at all
    got = verify_drafts(x, drafts, u)
    assert got.tokens[:, 1].tolist() == [4096] * B


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_verify_strides_and_addresses(dtype, dev):
    """Views of wider tensors at every offset from a 16-byte boundary, transposed
    batches and a transposed vocabulary give the dense call's tokens."""
    from naylis_amd.mom_kernels import verify_drafts
    c = _case(5, 3, 2501, dtype, dtype, dev)
    x, q = c["logits"], c["draft_probs"]
    run = lambda x, q: verify_drafts(x, c["drafts"], c["uniforms"], draft_probs=q)  # noqa: E731
    want = run(x, q)
    wide_x, wide_q = (torch.zeros(*t.shape[:2], 2520, dtype=dtype, device=dev) for t in (x, q))
    for off in range(9):
        wide_x[..., off:off + 2501], wide_q[..., 8 - off:2509 - off] = x, q
        got = run(wide_x[..., off:off + 2501], wide_q[..., 8 - off:2509 - off])
        assert torch.equal(got.tokens, want.tokens)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, q)]
    assert torch.equal(run(*turned).tokens, want.tokens)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, q)]
    assert torch.equal(run(*turned).tokens, want.tokens)
    same = run(x[:1].expand(5, -1, -1), q[:1].expand(5, -1, -1))
    one = verify_drafts(x[:1], c["drafts"][:1], c["uniforms"][:1], draft_probs=q[:1])
    assert torch.equal(same.tokens[:1], one.tokens)


@pytest.mark.parametrize("probs", [True, False])
def test_verified_tokens_are_the_models_own(probs, dev):
    """First tokens of 200000 sequences: whatever drew the drafts, each token comes
    as often as p says, within five standard deviations of a binomial count."""
    from naylis_amd.mom_kernels import verify_drafts
    g = torch.Generator(device=dev).manual_seed(11)
    V, B = 12, 50000
    x = torch.randn(1, 1, V, generator=g, device=dev) * 1.5
    q = torch.softmax(torch.randn(V, generator=g, device=dev), 0)
    counts = torch.zeros(V, device=dev)
    for _ in range(4):
        drafts = torch.multinomial(q, B, replacement=True, generator=g)[:, None] if probs else torch.full((B, 1), 3, device=dev)
        r = verify_drafts(x.expand(B, 2, V), drafts, torch.rand(B, 2, generator=g, device=dev),
                          draft_probs=q.expand(B, 1, V) if probs else None)
        counts += torch.bincount(r.tokens[:, 0], minlength=V)
    p = torch.softmax(x[0, 0].double(), 0)
    n = 4 * B
    assert bool(((counts.double() - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all())


def test_verify_streams_and_graph(dev):
    """Another stream, and two captured calls replayed on new logits, drafts,
    lengths and random numbers with eager calls between."""
    from naylis_amd.mom_kernels import verify_drafts
    c = _case(7, 3, 9001, torch.bfloat16, torch.float32, dev)
    lens, temps = torch.full((7,), 3, dtype=torch.int32, device=dev), torch.ones(7, device=dev)
    run = lambda: verify_drafts(c["logits"], c["drafts"], c["uniforms"], draft_probs=c["draft_probs"], draft_lens=lens,  # noqa: E731
                                temperature=temps)
    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    assert torch.equal(got.tokens, want.tokens)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run()
        graphs.append((graph, out))
    for i in range(6):
        new = _case(7, 3, 9001, torch.bfloat16, torch.float32, dev, seed=i + 1)
        for n in c:
            c[n].copy_(new[n])
        lens.copy_(torch.tensor([(i + j) % 4 for j in range(7)], dtype=torch.int32))
        temps[i] = 0.0
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        assert torch.equal(out.tokens, eager.tokens) and torch.equal(out.accepted, eager.accepted)


def test_verify_large_logits(dev):
    """Rows past 2^31 elements."""
    from naylis_amd.mom_kernels import verify_drafts
    B, N, V = 4, 15, 36000000
    x = torch.zeros(B, N + 1, V, dtype=torch.bfloat16, device=dev)
    for b in range(B):
        for i in range(N + 1):
            x[b, i, 35999000 + 17 * b + i] = 40.0  # all of p but 2^-32 or so
    want = torch.tensor([[35999000 + 17 * b + i for i in range(N + 1)] for b in range(B)], device=dev)
    u = torch.full((B, N + 1), 0.5, device=dev)
    got = verify_drafts(x, want[:, :N], u)
    assert torch.equal(got.tokens, want) and got.accepted.tolist() == [N] * B
    drafts = want[:, :N].clone()
    drafts[:, 9] = 5
    got = verify_drafts(x, drafts, u)
    assert got.accepted.tolist() == [9] * B and torch.equal(got.tokens[:, :10], want[:, :10])


@pytest.mark.parametrize("probs", [False, True], ids=["rule", "q32"])
@pytest.mark.parametrize("V", [700, 26001])  # one launch, three
def test_verify_most_sequences(V, probs, dev):
    """65535 sequences with a draft each (the most of a call), one row of logits for all."""
    from naylis_amd.mom_kernels import verify_drafts
    B = 65535
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.randn(1, 1, V, generator=g, device=dev) * 2
    p = torch.softmax(x[0, 0].double(), 0)
    q = torch.softmax(torch.randn(V, generator=g, device=dev) * 2, 0)
    d = torch.multinomial(q, B, replacement=True, generator=g)
    u = torch.rand(B, 2, generator=g, device=dev)
    got = verify_drafts(x.expand(B, 2, V), d[:, None], u, draft_probs=q.expand(B, 1, V) if probs else None)
    left = u[:, 0].double() * (q[d].double() if probs else 1.0) - p[d]
    kept = left < 0
    # p and p behind kept drafts; what is left of p, or p without the draft, behind others
    place = lambda cum, target: torch.searchsorted(cum, target[:, None], right=True).clamp(max=V - 1)[:, 0]  # noqa: E731
    cum, t = p.cumsum(0), u[:, 1].double()
    want = place(cum, t * cum[-1])
    near = (left.abs() < 2.0 ** -20 * p[d]) | ((cum[want] - t).abs() < 2.0 ** -38)
    if probs:
        rest = (p - q.double()).clamp(min=0).cumsum(0)
        other = place(rest, t * rest[-1])
        edge = (rest[other] / rest[-1] - t).abs().minimum((rest[(other - 1).clamp(min=0)] / rest[-1] - t).abs())
    else:
        # tokens below the draft have their cumulative weight, those above it p[d] less
        target = t * (cum[-1] - p[d])
        before = place(cum, target)
        other = torch.where(before < d, before, place(cum, target + p[d]))
        edge = (cum[other] - target - torch.where(before < d, 0.0, p[d])).abs()
    near |= (cum[(want - 1).clamp(min=0)] - t).abs() < 2.0 ** -38
    near |= edge < 2.0 ** -38
    assert int(near.sum()) < 100, "the inputs put random numbers next to borders"
    assert torch.equal(got.accepted.bool()[~near], kept[~near])
    first, second = torch.where(kept, d, other), torch.where(kept, want, -1)
    assert torch.equal(got.tokens[~near], torch.stack((first, second), 1)[~near])


def test_verify_refusals(dev):
    from naylis_amd.mom_kernels import verify_drafts
    c = _case(3, 2, 50, torch.float32, torch.float32, dev)
    x, d, u, q = c["logits"], c["drafts"], c["uniforms"], c["draft_probs"]
    bad = [(x[0], d, u), (x.half(), d, u), (x[:, :2], d, u), (x[..., :0], d, u), (x[:, :0], d[:, :0], u[:, :0]), (x, d.float(), u),
           (x, d[:2], u), (x, d, u[:, :2]), (x, d, u.double()), (x, d.cpu(), u), (x, d, u.cpu()), (x.cpu(), d, u)]
    for args in bad:
        with pytest.raises(RuntimeError, match="verify_drafts"):
            verify_drafts(*args)
    for kw in (dict(draft_probs=q[:, :1]), dict(draft_probs=q.half()), dict(draft_probs=q[..., :49]), dict(draft_probs=q.cpu()),
               dict(draft_lens=d), dict(draft_lens=u[:, 0]), dict(temperature=u), dict(temperature=d[:, 0]),
               dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(temperature=u[:2, 0])):
        with pytest.raises(RuntimeError, match="verify_drafts"):
            verify_drafts(x, d, u, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        verify_drafts(x.clone().requires_grad_(), d, u)
    r = verify_drafts(x[:0], d[:0], u[:0])
    assert r.tokens.shape == (0, 3) and r.accepted.shape == (0,)

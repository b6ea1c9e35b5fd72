"""packed_attention (naylis_mom_packed_attn_*) against fp64 attention of each
sequence on the same bf16 inputs: lengths around the tiles (32-row products,
64-row stages, 128-row workgroups), empty sequences, queries without keys, keys
of earlier tokens, grouped heads, heads of 64 and 128, rows outside every
sequence, more sequences than one wave's lanes."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

# query lengths, key lengths (None: the same), H, Hkv, hd, rows outside before and behind
CASES = [
    ([1], None, 1, 1, 64, 0, 0),
    ([1], [1], 2, 1, 128, 0, 0),
    ([31, 1, 0, 33], None, 2, 1, 64, 0, 0),
    ([64, 65, 127, 129], None, 4, 2, 128, 3, 200),
    ([5, 200, 40], [0, 131, 40], 4, 1, 64, 0, 5),       # no keys at all; queries before the first key
    ([150, 0, 7], [20, 90, 7], 4, 4, 128, 1, 1),
    ([257, 3, 300], [700, 3, 513], 8, 8, 128, 0, 0),
    ([1, 1, 1, 64], [1000, 64, 65, 128], 8, 2, 64, 0, 0),  # single new tokens after a cached prompt
    ([1021], None, 6, 3, 64, 0, 0),
    ([700], [2100], 6, 3, 128, 0, 0),
    ([2048, 999], None, 32, 8, 64, 0, 0),
    ([1537, 130], None, 16, 2, 128, 0, 130),
    ([900, 1500], None, 32, 8, 128, 0, 0),              # grids that fill the chip: whole tiles a workgroup
    ([1500], None, 64, 64, 64, 0, 3),
    ([1500], [1600], 64, 64, 128, 0, 3),
    ([(7 * i) % 150 for i in range(70)], None, 4, 2, 64, 10, 10),
    ([(11 * i) % 40 for i in range(130)], [(11 * i) % 40 + (i % 3) * 50 for i in range(130)], 2, 1, 128, 0, 0),
]


def _inputs(lq, lk, H, Hkv, hd, head, tail, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + len(lq) + H)
    lk = lq if lk is None else lk
    T, Tk = head + sum(lq) + tail, tail + sum(lk) + head
    q, d = (torch.randn(T, H, hd, generator=g, device=dev) for _ in range(2))
    k, v = (torch.randn(Tk, Hkv, hd, generator=g, device=dev) for _ in range(2))
    q[T // 2:] *= 5  # sharp rows: the running maximum has to move
    cq = torch.tensor([head] + [head + sum(lq[:i + 1]) for i in range(len(lq))], dtype=torch.int32, device=dev)
    ck = torch.tensor([tail] + [tail + sum(lk[:i + 1]) for i in range(len(lk))], dtype=torch.int32, device=dev)
    return [t.bfloat16() for t in (q, k, v, d)] + [cq, ck]


def _reference(q, k, v, d, cq, ck, scale):
    """fp64 results and, for each, what bounds its error: a bf16 rounding is at
    most 2^-8 relative, P (or dS) and the result are rounded once each, which
    is 2^-7 of the sum of the terms' magnitudes; delta reads the rounded output,
    whose error is 2^-8 of sum |dO| |o|, inside the 2^-7 too.  fp32 sums of at
    most 4096 terms and exponents of scores under 2^9 add less than 2^-10."""
    H, Hkv = q.shape[1], k.shape[1]
    G = H // Hkv
    shapes = {"o": q, "dq": q, "dk": k, "dv": v}
    res = {n: (torch.zeros(t.shape, dtype=torch.float64, device=q.device),
               torch.zeros(t.shape, dtype=torch.float64, device=q.device)) for n, t in shapes.items()}
    cq, ck = cq.tolist(), ck.tolist()
    for a, b, e, f in zip(cq, cq[1:], ck, ck[1:]):
        lq, lk = b - a, f - e
        if lq == 0 or lk == 0:
            continue
        see = torch.ones(lq, lk, dtype=torch.bool, device=q.device).tril(lk - lq)
        for h in range(H):
            x, dx = q[a:b, h].double(), d[a:b, h].double()
            y, z = k[e:f, h // G].double(), v[e:f, h // G].double()
            p = torch.softmax((x @ y.T * scale).masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
            o = p @ z
            dp = dx @ z.T
            delta = (dx * o).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            ads = p * (dp.abs() + delta.abs() + (dx.abs() * o.abs()).sum(-1, keepdim=True)) * scale
            for n, at, want, size in (("o", (slice(a, b), h), o, p @ z.abs()), ("dq", (slice(a, b), h), ds @ y, ads @ y.abs()),
                                      ("dk", (slice(e, f), h // G), ds.T @ x, ads.T @ x.abs()),
                                      ("dv", (slice(e, f), h // G), p.T @ dx, p.T @ dx.abs())):
                res[n][0][at] += want
                res[n][1][at] += size
    return {n: (w, s * (2.0 ** -7 + 2.0 ** -10)) for n, (w, s) in res.items()}


def _run(q, k, v, d, cq, ck, scale):
    from naylis_amd.mom_kernels import packed_attention
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = packed_attention(q, k, v, cq, ck, scale=scale)
    grads = torch.autograd.grad(o, (q, k, v), d)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))


def _check(got, want):
    for n, (w, bound) in want.items():
        err = (got[n].double() - w).abs()
        assert bool((err <= bound + 1e-30).all()), (n, float((err / (bound + 1e-30)).max()))


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}seqs-{sum(c[0])}-H{c[2]}/{c[3]}x{c[4]}")
def test_packed_matches_fp64(case, dev):
    x = _inputs(*case, dev)
    scale = case[4] ** -0.5
    got = _run(*x, scale)
    _check(got, _reference(*x, scale))
    from naylis_amd.mom_kernels import packed_attention
    with torch.no_grad():  # the call without a gradient gives the same
        assert torch.equal(packed_attention(*x[:3], *x[4:]), got["o"])


def test_packed_gradient_matches_differences(dev):
    """The gradient along a direction against a difference quotient of the fp64
    formula at the kernel's own inputs."""
    x = _inputs([40, 17], [55, 17], 4, 2, 64, 0, 0, dev)
    q, k, v, d, cq, ck = x
    got = _run(*x, 0.125)
    g = torch.Generator(device=dev).manual_seed(5)

    def value(q, k, v):
        total = 0.0
        for a, b, e, f in zip(cq.tolist(), cq.tolist()[1:], ck.tolist(), ck.tolist()[1:]):
            see = torch.ones(b - a, f - e, dtype=torch.bool, device=dev).tril(f - e - b + a)
            for h in range(4):
                s = (q[a:b, h] @ k[e:f, h // 2].T * 0.125).masked_fill(~see, -math.inf)
                total = total + ((torch.softmax(s, -1) @ v[e:f, h // 2]) * d[a:b, h].double()).sum()
        return total

    for i, n in enumerate(("dq", "dk", "dv")):
        u = torch.randn(x[i].shape, generator=g, device=dev, dtype=torch.float64)
        lo, hi = ([t.double() + (s * 1e-4 * u if j == i else 0) for j, t in enumerate((q, k, v))] for s in (-1, 1))
        slope = float(value(*hi) - value(*lo)) / 2e-4
        w, bound = _reference(*x, 0.125)[n]
        assert abs(float((got[n].double() * u).sum()) - slope) <= float((bound * u.abs()).sum()) + 1e-5 * abs(slope)


def test_packed_sequences_do_not_see_each_other(dev):
    """Garbage in one sequence reaches no other, bit for bit, and neither does
    what stands outside the sequences; runs repeat bit for bit."""
    x = _inputs([70, 130, 45], [70, 190, 45], 4, 2, 128, 5, 9, dev)
    a = _run(*x, 0.1)
    b = _run(*x, 0.1)
    assert all(torch.equal(a[n], b[n]) for n in a)
    y = [t.clone() for t in x]
    cq, ck = x[4].tolist(), x[5].tolist()
    for t, c in ((y[0], cq), (y[3], cq), (y[1], ck), (y[2], ck)):
        t[c[1]:c[2]] = math.nan
        t[:c[0]] = math.inf
        t[c[3]:] = math.nan
    c = _run(*y, 0.1)
    for n, off in (("o", cq), ("dq", cq), ("dk", ck), ("dv", ck)):
        for s in (slice(0, off[1]), slice(off[2], None)):
            assert torch.equal(a[n][s], c[n][s]), n
    assert bool((a["o"][:5] == 0).all() and (a["dk"][ck[3]:] == 0).all() and (a["dv"][:ck[0]] == 0).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("top", [4.0, 30.0])
def test_packed_rising_scores(top, hd, dev):
    """Scores that grow or fall along the keys by a little or a lot a tile."""
    q, k, v, d, cq, ck = _inputs([300, 300], [420, 420], 4, 2, hd, 0, 0, dev)
    one = torch.ones(hd, device=dev)
    ramp = torch.linspace(0, top, 420, device=dev)
    k = (k.float() * 0.1 + torch.cat([ramp, ramp.flip(0)])[:, None, None] * one / hd ** 0.5).bfloat16()
    q = (q.float() * 0.1 + one).bfloat16()
    x = (q, k, v, d, cq, ck)
    _check(_run(*x, 0.7), _reference(*x, 0.7))


@pytest.mark.parametrize("n,longest", [(22, 200), (23, 200), (63, 90), (4200, 3)])
def test_packed_many_sequences(n, longest, dev):
    """Either side of the count from which sequences are taken in their order,
    and more than a search of two rounds covers; empty ones among them."""
    r = random.Random(n)
    lq = [r.choice([0, 1, r.randint(0, longest)]) for _ in range(n)]
    lk = [a + r.choice([0, r.randint(0, longest)]) for a in lq]
    x = _inputs(lq, lk, 2, 1, 64, 3, 140, dev)
    _check(_run(*x, 0.125), _reference(*x, 0.125))


def test_packed_is_causal(dev):
    x = _inputs([333], [400], 4, 4, 64, 0, 0, dev)
    y = [t.clone() for t in x]
    for t in y[1:3]:
        t[267:] *= 7  # keys behind query 199's last
    assert torch.equal(_run(*x, 0.125)["o"][:200], _run(*y, 0.125)["o"][:200])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shift", [0, 5, 31])
def test_packed_garbage_stays_near(shift, hd, dev):
    """A NaN in a row of v or k reaches, beside the queries that see it, at most
    62 queries before them (k: none); one in dO at most 62 keys behind it."""
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, cq, ck = _inputs([300], [300 + shift], 4, 2, hd, 0, 0, dev)
    want = _run(q, k, v, d, cq, ck, 0.1)
    for row in (64, 161, 200):
        bad = [t.clone() for t in (q, k, v, d)]
        bad[2][row] = math.nan
        o = packed_attention(*bad[:3], cq, ck, scale=0.1)
        first = row - shift  # the first query that sees it
        assert torch.equal(o[:max(first - 62, 0)], want["o"][:max(first - 62, 0)]) and bool(o[first:].isnan().all())
        bad[2], bad[1][row] = v, math.nan
        o = packed_attention(*bad[:3], cq, ck, scale=0.1)
        assert torch.equal(o[:first], want["o"][:first]) and bool(o[first:].isnan().all())
        bad[1], bad[3][row] = k, math.nan
        dv = _run(*bad, cq, ck, 0.1)["dv"]
        last = row + shift  # the last key that it sees
        assert torch.equal(dv[last + 63:], want["dv"][last + 63:]) and bool(dv[:last + 1].isnan().all())


def _far_inputs(size, sign, lens, H, Hkv, hd, dev):
    """Scores of up to size^2 / 8 either way, each of few values (equal ones equal
    bit for bit, others far apart), and queries so small that theirs are ordinary."""
    q, k, v, d, cq, ck = _inputs(*lens, H, Hkv, hd, 0, 0, dev)
    i, j = (torch.arange(t.shape[0], device=dev)[:, None] for t in (q, k))
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[..., 3] = torch.where(i % 3 == 0, 2.0 ** -6 / size, size * 2.0 ** -(i % 2))
    grade = torch.where((j * 5) % 13 == 0, 4.0, 2.0) * torch.where(j < 70, 0.25, 1.0)  # rises within a walk
    k[..., 3] = sign * size / 4 * (grade if sign > 0 else 5 - grade)
    return q, k, v, d, cq, ck


FAR = [2.0 ** 10, 2.0 ** 17, 2.0 ** 30, 2.0 ** 60]
FAR_LENS = [([300, 1, 33], None), ([90, 200], [400, 260]), ([40], [20])]


@pytest.mark.parametrize("hd,H", [(64, 4), (128, 4), (64, 600), (128, 400)])  # two waves for 32 queries, and one
@pytest.mark.parametrize("lens", FAR_LENS, ids=["same", "earlier", "none"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", FAR)
def test_packed_scores_of_any_size(size, sign, lens, hd, H, dev):
    """Weights of far scores are 0 or equal ones; the bounds are the ordinary ones."""
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, cq, ck = _far_inputs(size, sign, lens, 4, 2, hd, dev)
    want = _reference(q, k, v, d, cq, ck, 0.125)["o"]
    wide = lambda t: t.repeat(1, H // 4, 1)  # noqa: E731
    heads = torch.arange(H, device=dev) % 2 if H > 4 else torch.arange(2, device=dev)
    o = packed_attention(wide(q), k[:, heads], v[:, heads], cq, ck, scale=0.125)
    for h in range(0, H, max(H // 8, 1)):
        kv = int(heads[h]) if H > 4 else h // 2
        err = (o[:, h].double() - want[0][:, 2 * kv]).abs()
        assert bool((err <= want[1][:, 2 * kv] + 1e-30).all()), (h, float(err.max()))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 16, 2.0 ** 30])
def test_packed_far_random_scores(size, hd, dev):
    """Random far scores: where a query's highest lies clear of the next one by
    more than fp32 sums of hd products may be off, its result is that key's v (within
    the roundings of P and of the result); an
    ordinary query's does not depend on its far neighbours, bit for bit."""
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, cq, ck = _inputs([200, 130], [350, 130], 4, 2, hd, 0, 0, dev)
    usual = packed_attention(q, k, v, cq, ck)
    far = torch.arange(330, device=dev) % 5 != 0
    q = torch.where(far[:, None, None], q * size * size, q)
    o = packed_attention(q, k, v, cq, ck)
    assert bool(o.isfinite().all()) and torch.equal(o[~far], usual[~far])
    clear = 0
    for a, b, e, f in ((0, 200, 0, 350), (200, 330, 350, 480)):
        see = torch.ones(b - a, f - e, dtype=torch.bool, device=dev).tril(f - e - b + a)
        for h in range(4):
            x, y = q[a:b, h].double(), k[e:f, h // 2].double()
            s = (x @ y.T * hd ** -0.5).masked_fill(~see, -math.inf)
            noise = (x.abs() @ y.abs().T * hd ** -0.5).amax(-1) * hd * 2.0 ** -23
            top, at = s.topk(2, -1)
            sure = far[a:b] & (top[:, 0] - top[:, 1] > 2 * noise + 40)
            clear += int(sure.sum())
            best = v[e:f, h // 2][at[sure, 0]].double()  # (times P / l, whose P is rounded to bf16, and rounded once)
            assert bool(((o[a:b, h][sure].double() - best).abs() <= best.abs() * (2.0 ** -7 + 2.0 ** -10)).all())
    assert clear > 300


@pytest.mark.parametrize("hd,copies", [(64, 1), (128, 1), (64, 150), (128, 100)])  # pairs of waves, and tiles a wave
@pytest.mark.parametrize("lens", FAR_LENS, ids=["same", "earlier", "none"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", [2.0 ** 6, 2.0 ** 8] + FAR)
def test_packed_gradients_of_scores_of_any_size(size, sign, lens, hd, copies, dev):
    """The ordinary bounds, for ordinary queries and far ones among each other; a
    far query's weights are 0 or equal ones.  Copies of the heads give the same bits."""
    H, Hkv = (4, 2) if copies == 1 else (2, 2)
    x = _far_inputs(size, sign, lens, H, Hkv, hd, dev)
    want = _reference(*x, 0.125)
    got = _run(*(t.repeat(1, copies, 1) for t in x[:4]), *x[4:], 0.125)
    if copies > 1:
        for n, t in got.items():
            parts = t.view(t.shape[0], copies, -1, hd)
            assert torch.equal(parts, parts[:, :1].expand_as(parts)), n
            got[n] = parts[:, 0]
    _check(got, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 30])
def test_packed_far_scores_in_parts_and_views(size, hd, dev):
    """A group's heads in parts (few key tiles, many heads), rows outside the
    sequences, operands of any stride, an expanded gradient: the bits of dense ones."""
    q, k, v, d, cq, ck = _far_inputs(size, 1, ([700, 260], [900, 260]), 8, 2, hd, dev)
    edge = lambda t: torch.cat([t[:7], t, t[:50]])  # noqa: E731
    x = [edge(t) for t in (q, k, v, d)] + [cq + 7, ck + 7]
    got = _run(*x, 0.125)
    _check(got, _reference(*x, 0.125))
    assert all(torch.equal(a, b) for a, b in zip(got.values(), _run(*x, 0.125).values()))
    wide = torch.cat([x[0].flatten(1), x[3].flatten(1)], 1)
    views = [wide[:, :8 * hd].view(-1, 8, hd), x[1].transpose(0, 1).contiguous().transpose(0, 1),
             torch.cat([x[2], x[2]], 2)[..., hd:], wide[:, -8 * hd:].view(-1, 8, hd)]
    assert all(torch.equal(a, b) for a, b in zip(got.values(), _run(*views, *x[4:], 0.125).values()))
    ones = torch.ones(1, 1, 1, dtype=q.dtype, device=dev).expand_as(x[0])
    same = _run(*x[:3], torch.ones_like(x[3]), *x[4:], 0.125)
    assert all(torch.equal(a, b) for a, b in zip(same.values(), _run(*x[:3], ones, *x[4:], 0.125).values()))


@pytest.mark.parametrize("hd,H,Hkv", [(64, 4, 2), (128, 4, 2), (64, 300, 300), (128, 200, 200)])
@pytest.mark.parametrize("size", [2.0 ** 6, 2.0 ** 16, 2.0 ** 30])
def test_packed_gradients_of_far_random_scores(size, hd, H, Hkv, dev):
    """Random far scores: queries whose highest lies clear of the next by more than
    fp32 sums may be off are one key's each (the others get no gradient); ordinary
    queries' dq, and with far queries' dO zero all of dk and dv, do not depend on
    the far ones, bit for bit."""
    q, k, v, d, cq, ck = _inputs([200, 130], [350, 130], 4, 2, hd, 0, 0, dev)
    q, d = (t.repeat(1, H // 4, 1) for t in (q, d))
    k, v = (t.repeat(1, Hkv // 2, 1) for t in (k, v))
    far = (torch.arange(330, device=dev) % 5 != 0)[:, None, None]
    scale = hd ** -0.5
    usual = _run(q, k, v, d.masked_fill(far, 0.0), cq, ck, scale)
    q = torch.where(far, q * size * size, q)
    none = _run(q, k, v, d.masked_fill(far, 0.0), cq, ck, scale)
    assert torch.equal(none["dk"], usual["dk"]) and torch.equal(none["dv"], usual["dv"])
    if H > 4:  # (the reference goes head by head)
        q, d = (t[:, :4].contiguous() for t in (q, d))
        k, v = (t[:, :4].contiguous() for t in (k, v))
    G, clear = q.shape[1] // k.shape[1], 0
    for a, b, e, f in ((0, 200, 0, 350), (200, 330, 350, 480)):
        see = torch.ones(b - a, f - e, dtype=torch.bool, device=dev).tril(f - e - b + a)
        for h in range(4):
            x, y = q[a:b, h].double(), k[e:f, h // G].double()
            top = (x @ y.T * scale).masked_fill(~see, -math.inf).topk(2, -1)[0]
            noise = (x.abs() @ y.abs().T * scale).amax(-1) * hd * 2.0 ** -23
            sure = (top[:, 0] - top[:, 1] > 2 * noise + 40) | ~far[a:b, 0, 0]
            clear += int(sure.sum())
            d[a:b, h] = torch.where(sure[:, None], d[a:b, h], 0.0)
    assert clear > 600
    want = _reference(q, k, v, d, cq, ck, scale)
    if H > 4:
        q, k, v, d = (t.repeat(1, H // 4, 1) for t in (q, k, v, d))
    got = _run(q, k, v, d, cq, ck, scale)
    plain = ~far[:, 0, 0]
    assert torch.equal(got["dq"][plain], usual["dq"][plain])
    # o of the queries that are not clear is not the reference's
    _check({n: t[:, :want[n][0].shape[1]] for n, t in got.items() if n != "o"}, {n: w for n, w in want.items() if n != "o"})


@pytest.mark.parametrize("hd,copies", [(64, 1), (128, 1), (64, 150), (128, 100)])
@pytest.mark.parametrize("shift", [0, 5, 31])
def test_packed_garbage_stays_near_in_the_gradients(shift, hd, copies, dev):
    """A NaN in a row of k or v reaches, beside dq of the queries that see it, that of
    at most 62 before them; one in q or dO, beside dk of the keys that its query
    sees, that of at most 62 behind them, and one in q no further key's dv."""
    H = 4 * copies
    q, k, v, d, cq, ck = _inputs([300], [300 + shift], H, H // 2, hd, 0, 0, dev)
    want = _run(q, k, v, d, cq, ck, 0.1)
    for row in (64, 161, 200):
        first, last = row - shift, row + shift  # the first query that sees the key, the last key that the query sees
        for i in (1, 2):
            bad = [t.clone() if j == i else t for j, t in enumerate((q, k, v, d))]
            bad[i][row] = math.nan
            dq = _run(*bad, cq, ck, 0.1)["dq"]
            near = max(first - 62, 0)
            assert torch.equal(dq[:near], want["dq"][:near]) and bool(dq[first:].isnan().all())
        for i in (0, 3):
            bad = [t.clone() if j == i else t for j, t in enumerate((q, k, v, d))]
            bad[i][row] = math.nan
            got = _run(*bad, cq, ck, 0.1)
            assert torch.equal(got["dk"][last + 63:], want["dk"][last + 63:]) and bool(got["dk"][:last + 1].isnan().all())
            assert torch.equal(got["dq"][:row], want["dq"][:row]) and torch.equal(got["dq"][row + 1:], want["dq"][row + 1:])
            if i == 0:
                assert torch.equal(got["dv"][last + 1:], want["dv"][last + 1:]) and bool(got["dv"][:last + 1].isnan().all())


@pytest.mark.parametrize("hd,H", [(64, 4), (128, 4), (64, 600), (128, 400)])
@pytest.mark.parametrize("bad", ["k", "v"])
def test_packed_queries_without_keys_are_zero(bad, hd, H, dev):
    """Whatever the sequence's keys and values hold, a query that sees none of them
    gives 0 and has a gradient of 0."""
    x = _inputs([90, 40], [30, 33], H, H // 2, hd, 0, 0, dev)
    for value in (math.nan, math.inf):
        t = x[1 if bad == "k" else 2]
        t[3] = t[35] = value
        got = _run(*x, 0.125)
        for n in ("o", "dq"):
            assert bool((got[n][:60] == 0).all() and (got[n][90:97] == 0).all()), n
            assert not bool(got[n][60:90].isfinite().all())


def test_packed_equals_the_batch_kernel(dev):
    """Equal lengths and heads of 64: the framework's batch attention within
    both kernels' bounds."""
    from naylis_amd.mom_kernels import packed_attention
    from naylis_amd.mom_kernels.hip_attention import causal_attention
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v = (torch.randn(3, 200, 4, 64, generator=g, device=dev).bfloat16() for _ in range(3))
    cu = torch.arange(0, 601, 200, dtype=torch.int32, device=dev)
    got = packed_attention(*(t.view(600, 4, 64) for t in (q, k, v)), cu).view(3, 200, 4, 64)
    want = causal_attention(q, k, v, 0.125)
    assert float((got.float() - want.float()).norm() / want.float().norm()) < 2.0 ** -7


def test_packed_takes_views(dev):
    """q, k, v as slices of one projection, gradients of strided and expanded
    outputs, int64 offsets, and unaligned or feature-strided operands (copied)."""
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, cq, ck = _inputs([90, 41], None, 4, 2, 64, 0, 0, dev)
    want = _run(q, k, v, d, cq, ck, 0.125)
    qkv = torch.cat([t.flatten(1) for t in (q, k, v)], 1).requires_grad_()
    a, b, c = (t.view(131, -1, 64) for t in qkv.split([256, 128, 128], 1))
    o = packed_attention(a, b, c, cq.long())
    assert torch.equal(o, want["o"])
    dd = torch.cat([d, d], 2)[..., 64:]  # strided gradient
    grad, = torch.autograd.grad(o, qkv, dd)
    assert torch.equal(grad, torch.cat([want[n].flatten(1) for n in ("dq", "dk", "dv")], 1))
    ones = _run(q, k, v, torch.ones_like(d), cq, ck, 0.125)
    x, y, z = (t.clone().requires_grad_() for t in (q, k, v))
    packed_attention(x, y, z, cq).sum().backward()  # an expanded gradient
    assert all(torch.equal(t.grad, ones[n]) for t, n in ((x, "dq"), (y, "dk"), (z, "dv")))
    for make in (lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape),  # not 16-byte aligned
                 lambda t: t.permute(2, 0, 1).contiguous().permute(1, 2, 0),   # features not dense
                 lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):    # heads outermost
        assert torch.equal(packed_attention(make(q), make(k), make(v), cq), want["o"])


def test_packed_single_rows_and_heads(dev):
    """One token, or one head, of a wider tensor whose strides are no whole
    16-byte pieces (torch takes any stride of a single row for dense)."""
    from naylis_amd.mom_kernels import packed_attention
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(3, 643, generator=g, device=dev).bfloat16()
    q, k, v = (torch.as_strided(x, (1, 2, 64), (643, 64, 1), 128 * i) for i in range(3))
    assert q.is_contiguous() and q.stride(0) % 8 != 0
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    assert torch.equal(packed_attention(q, k, v, cu), v)
    y = torch.randn(5, 3, 64, generator=g, device=dev).bfloat16()
    q, k, v = (torch.as_strided(y, (5, 1, 64), (192, 7, 1), 64 * i) for i in range(3))
    cu = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    assert torch.equal(packed_attention(q, k, v, cu), packed_attention(*(t.clone() for t in (q, k, v)), cu))


def test_packed_far_rows(dev):
    """Rows and heads further than 2^32 bytes from the tensor's start."""
    T, ld = 290, (1 << 23) - 8
    q, k, v, d, cq, ck = _inputs([T], None, 4, 2, 64, 0, 0, dev)
    want = _run(q, k, v, d, cq, ck, 0.125)
    room = torch.empty(T * ld + 64, dtype=torch.bfloat16, device=dev)
    far = [torch.as_strided(room, t.shape, (ld, 1 << 20, 1), at) for t, at in ((q, 0), (k, 64), (v, 128), (d, 192))]
    for f, t in zip(far, (q, k, v, d)):
        f.copy_(t)
    got = _run(*far, cq, ck, 0.125)
    assert all(torch.equal(got[n], want[n]) for n in got)
    step = room.numel() // 4 // 192 * 192
    for i, t in enumerate((q, k, v)):  # heads outermost
        far[i] = torch.as_strided(room, t.shape, (192, 4 // t.size(1) * step, 1), 64 * i).copy_(t)
    got = _run(*far[:3], d, cq, ck, 0.125)
    assert all(torch.equal(got[n], want[n]) for n in got)


def test_packed_large_tensors(dev):
    """Queries, results and gradients of more than 2^31 elements."""
    n, L, H = 16400, 64, 32
    q, k, v, d, _, _ = _inputs([L] * 3, None, H, 1, 64, 0, 0, dev)
    cu = torch.arange(0, n * L + 1, L, dtype=torch.int32, device=dev)
    want = _reference(q, k, v, d, cu[:4], cu[:4], 0.125)
    x = [torch.zeros(n * L, *t.shape[1:], dtype=t.dtype, device=dev) for t in (q, k, v, d)]
    assert x[0].numel() > 2 ** 31
    for big, small in zip(x, (q, k, v, d)):
        big[-3 * L:] = small
        big[:3 * L] = small
    got = _run(*x, cu, cu, 0.125)
    _check({name: t[:3 * L] for name, t in got.items()}, want)
    for name, t in got.items():
        assert torch.equal(t[:3 * L], t[-3 * L:]) and not bool(t[3 * L:-3 * L].any()), name


def test_packed_empty_tensors(dev):
    from naylis_amd.mom_kernels import packed_attention
    z = lambda n, h: torch.zeros(n, h, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)  # noqa: E731
    none, some = (torch.tensor(c, dtype=torch.int32, device=dev) for c in ([0, 0], [0, 9]))
    o = packed_attention(z(0, 4), z(0, 2), z(0, 2), none)
    assert o.shape == (0, 4, 64)
    q, k, v = z(9, 4), z(0, 2), z(0, 2)
    o = packed_attention(q, k, v, some, none)
    o.sum().backward()
    assert bool((o == 0).all() and (q.grad == 0).all()) and k.grad.shape == (0, 2, 64)
    q, k, v = z(0, 4), z(9, 2), z(9, 2)
    packed_attention(q, k, v, none, some).sum().backward()
    assert bool((k.grad == 0).all() and (v.grad == 0).all())


def test_packed_offsets_out_of_range_stay_inside(dev):
    """Offsets outside the tensors are clamped to them; descending ones leave
    rows unspecified and nothing else."""
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, _, _ = _inputs([200], None, 2, 2, 64, 0, 0, dev)
    c = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    want = packed_attention(q, k, v, c(0, 200))
    assert torch.equal(packed_attention(q, k, v, c(-5, 1 << 30)), want)
    rnd = random.Random(0)
    for _ in range(5):
        packed_attention(q, k, v, c(*(rnd.randint(-300, 500) for _ in range(6))),
                         c(*(rnd.randint(-300, 500) for _ in range(6))))
    torch.cuda.synchronize()
    assert torch.equal(packed_attention(q, k, v, c(0, 200)), want)


def test_packed_streams_and_graph(dev):
    """Another stream than the current one at creation, and a captured forward
    and backward replayed on new inputs and new offsets."""
    x = _inputs([100, 156], [130, 300], 4, 2, 128, 0, 0, dev)
    want = _run(*x, 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(*x, 0.1)
    s.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    held = [t.clone() for t in x]
    with torch.cuda.stream(s):
        _run(*held, 0.1)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs = _run(*held, 0.1)
    for lens in ([100, 156], [1, 255], [256, 0]):
        y = _inputs(lens, [130, 300], 4, 2, 128, 0, 0, dev, seed=lens[0])
        for a, b in zip(held, y):
            a.copy_(b)
        eager = _run(*y, 0.1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[n], eager[n]) for n in eager), lens


def test_packed_second_derivative_raises(dev):
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, cq, ck = _inputs([70], None, 2, 1, 64, 0, 0, dev)
    want = _run(q, k, v, d, cq, ck, 0.125)
    q, k, v, d = (t.requires_grad_() for t in (q, k, v, d))
    got = torch.autograd.grad(packed_attention(q, k, v, cq), (q, k, v), d, create_graph=True)
    assert all(torch.equal(a, want[n]) for a, n in zip(got, ("dq", "dk", "dv")))
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(got[0].float().sum(), k)


def test_packed_refusals(dev):
    from naylis_amd.mom_kernels import packed_attention
    q, k, v, d, cq, ck = _inputs([20], None, 4, 2, 64, 0, 0, dev)
    bad = [(q.float(), k, v, cq), (q[:, :3], k, v, cq), (q, k, v[:, :1], cq), (q[..., :32], k[..., :32], v[..., :32], cq),
           (q, k.cpu(), v, cq), (q, k, v, cq.cpu()), (q, k, v, cq.float()), (q, k, v, cq[:1]), (q[0], k, v, cq),
           (q, k[:, :0], v[:, :0], cq)]
    for args in bad:
        with pytest.raises(RuntimeError, match="packed_attention"):
            packed_attention(*args)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="scale"):
            packed_attention(q, k, v, cq, scale=scale)
    with pytest.raises(RuntimeError, match="packed_attention"):
        packed_attention(q, k, v, cq, torch.cat([ck, ck]))

"""Pages of 4 bits (e2m1 with a power of two for 32 features) and several new
tokens a sequence: paged_append and paged_attention against fp64 statements."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FORMATS = ("bf16", "e4m3", "e2m1")
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _cache(fmt, pages, Hkv, page, hd, dev):
    """Pages that hold NaN (or codes and scales of it) everywhere."""
    from naylis_amd.mom_kernels import PagedCache, new_paged_cache
    c = new_paged_cache(pages, Hkv, page, hd, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1")
    for t in c:
        if t is not None:
            t.fill_(math.nan if t.dtype.is_floating_point else 0x7f if fmt == "e4m3" else 0xff)
    return PagedCache(*c)


def _case(lens, H, Hkv, hd, page, fmt, dev, N=None, q_lens=None, width=None, seed=0):
    from naylis_amd.mom_kernels import paged_append
    g = torch.Generator(device=dev).manual_seed(seed + H + len(lens))
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    pages = sum(need) + 2
    ids = torch.randperm(pages, generator=g, device=dev).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    table = table.to(dev)
    T = sum(lens)
    k, v = (torch.randn(T, Hkv, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    shape = (len(lens), H, hd) if N is None else (len(lens), N, H, hd)
    q = (torch.randn(shape, generator=g, device=dev) * 2).bfloat16()
    rows = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(dev, torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev, torch.int32)
    cache = _cache(fmt, pages, Hkv, page, hd, dev)
    paged_append(cache, k, v, table, pos, rows)
    return dict(q=q, cache=cache, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev), k=k, v=v, rows=rows,
                pos=pos, q_lens=None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device=dev))


def _stored(c, page):
    """fp64 keys and values of the tokens, as the cache holds them."""
    at, off = c["table"][c["rows"].long(), c["pos"].long() // page].long(), c["pos"].long() % page
    return [x[at, :, off].double() for x in c["cache"].dequantize()]


def _attention(c, scale, page):
    """fp64 attention of each new token over what its sequence's cache holds, and
    what bounds the kernel's error: P (times a scale of e4m3 values) and the result
    are rounded to bf16 once each, at most 2^-8 relative; exponents and fp32 sums
    add less than 2^-10."""
    k, v = _stored(c, page)
    q = c["q"].double() if c["q"].dim() == 4 else c["q"].double()[:, None]
    B, N, H, _ = q.shape
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    G, at = H // k.shape[1], 0
    live = [N] * B if c["q_lens"] is None else [min(max(n, 0), N) for n in c["q_lens"].tolist()]
    for b, n in enumerate(c["lens"].tolist()):
        for i in range(live[b]):
            m = n - (live[b] - 1 - i)
            for h in range(H if m > 0 else 0):
                x, y = k[at:at + m, h // G], v[at:at + m, h // G]
                p = torch.softmax(x @ q[b, i, h] * scale, 0)
                out[b, i, h], size[b, i, h] = p @ y, p @ y.abs()
        at += n
    return out.view(c["q"].shape), (size * (2.0 ** -7 + 2.0 ** -10)).view(c["q"].shape)


def _check(c, page, scale=None):
    from naylis_amd.mom_kernels import paged_attention
    got = paged_attention(c["q"], c["cache"], c["table"], c["lens"], q_lens=c["q_lens"])
    want, bound = _attention(c, c["q"].shape[-1] ** -0.5, page)
    err = (got.double() - want).abs()
    assert bool((err <= bound + 1e-30).all()), float((err / (bound + 1e-30)).max())
    return got


# lengths, H, Hkv, hd, page
ONE = [
    ([1], 1, 1, 64, 16),
    ([1], 4, 1, 128, 16),
    ([0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 49], 4, 2, 64, 16),
    ([63, 0, 64, 65, 129, 0, 127, 128], 4, 4, 128, 32),
    ([500], 16, 16, 64, 16),
    ([5000, 3, 700, 0, 64], 8, 2, 128, 64),
    ([9001, 1, 1, 130], 8, 1, 64, 256),
    ([40, 300], 34, 2, 128, 128),                      # 17 query heads a key head
    ([(37 * i) % 400 for i in range(130)], 6, 2, 64, 32),
    ([70001], 4, 2, 128, 64),
    ([(53 * i) % 1900 for i in range(65)], 32, 8, 128, 16),
    ([(53 * i) % 1020 for i in range(65)], 8, 2, 128, 16),  # a workgroup for each, of more than 16 steps
    ([0] * 70 + [1600] + [0] * 200 + [(29 * i) % 90 for i in range(100)] + [0], 2, 1, 64, 16),
    ([0 if i % 3 else (i * i) % 23 for i in range(4200)] + [1530], 2, 1, 64, 16),  # chunks of 66 sequences
]


@pytest.mark.parametrize("case", ONE, ids=lambda c: f"B{len(c[0])}-{max(c[0])}-H{c[1]}/{c[2]}x{c[3]}-p{c[4]}")
def test_e2m1_matches_fp64(case, dev):
    c = _case(*case, "e2m1", dev)
    got = _check(c, case[4])
    from naylis_amd.mom_kernels import paged_attention
    assert torch.equal(got, paged_attention(c["q"], c["cache"], c["table"], c["lens"], scale=case[3] ** -0.5))


# lengths, H, Hkv, hd, page, N, q_lens
MANY = [
    ([1, 2, 3, 4, 5, 0], 4, 2, 64, 16, 4, None),                      # tokens that see nothing
    ([1, 9, 40, 16, 17, 33], 4, 2, 128, 16, 3, [1, 0, 3, 2, -5, 99]),
    ([300, 31, 32, 33, 64, 65], 8, 2, 64, 32, 5, [5, 4, 3, 2, 1, 5]),  # 20 rows a key head
    ([700, 64, 1], 8, 1, 128, 64, 9, [9, 7, 1]),                      # 72 rows
    ([5000, 3, 700, 0, 64], 8, 2, 128, 64, 2, None),                  # several workgroups a sequence
    ([2600, 1, 900], 4, 4, 64, 16, 8, [8, 8, 5]),
    ([40], 34, 2, 128, 128, 3, None),                                 # 51 rows, three products
    ([(53 * i) % 900 for i in range(65)], 8, 2, 64, 16, 4, [i % 5 for i in range(65)]),
    ([(53 * i) % 1900 for i in range(65)], 8, 2, 128, 16, 4, [i % 5 for i in range(65)]),
    ([(53 * i) % 1020 for i in range(35)], 16, 2, 128, 32, 5, [i % 6 for i in range(35)]),  # 40 rows, two slices
    ([600], 1, 1, 64, 16, 1, [1]),
    ([600, 20], 2, 1, 64, 16, 1, [0, 1]),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", MANY, ids=lambda c: f"B{len(c[0])}-{max(c[0])}-H{c[1]}/{c[2]}x{c[3]}-p{c[4]}-N{c[5]}")
def test_tokens_match_fp64(case, fmt, dev):
    """Each new token against the keys up to its own; rows behind a sequence's
    last one, and tokens that see nothing, are 0."""
    lens, H, Hkv, hd, page, N, q_lens = case
    c = _case(lens, H, Hkv, hd, page, fmt, dev, N=N, q_lens=q_lens)
    got = _check(c, page)
    live = [N] * len(lens) if q_lens is None else [min(max(n, 0), N) for n in q_lens]
    for b, n in enumerate(live):
        assert not bool(got[b, n:].any()) and not bool(got[b, :max(n - lens[b], 0)].any())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("width", [None, 100])  # a table of one launch, and of two
def test_tokens_of_one_are_the_single_form(fmt, width, dev):
    from naylis_amd.mom_kernels import paged_attention
    c = _case([20, 300, 0, 7], 8, 2, 64, 16, fmt, dev, width=width)
    want = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    for q_lens in (None, torch.ones(4, dtype=torch.int32, device=dev)):
        got = paged_attention(c["q"][:, None], c["cache"], c["table"], c["lens"], q_lens=q_lens)
        assert torch.equal(got[:, 0], want)
    got = paged_attention(c["q"], c["cache"], c["table"], c["lens"], q_lens=torch.ones(4, dtype=torch.int64, device=dev))
    assert torch.equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd", [64, 128])
def test_tokens_of_any_strides(fmt, hd, dev):
    """q as slices of a projection, token-major and head-major, and at odd addresses."""
    from naylis_amd.mom_kernels import paged_attention
    c = _case([70, 5, 333], 8, 2, hd, 16, fmt, dev, N=3, q_lens=[3, 2, 1])
    run = lambda q: paged_attention(q, c["cache"], c["table"], c["lens"], q_lens=c["q_lens"])  # noqa: E731
    q, want = c["q"], run(c["q"])
    assert torch.equal(run(q.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)), want)
    assert torch.equal(run(torch.cat([q, q], -2)[:, :, 8:]), want)
    assert torch.equal(run(torch.cat([q[..., :1], q], -1)[..., 1:]), want)
    assert torch.equal(run(q.transpose(-1, -2).contiguous().transpose(-1, -2)), want)
    assert torch.equal(run(q[:1].expand(3, -1, -1, -1))[0], want[0])


@pytest.mark.parametrize("fmt", FORMATS)
def test_tokens_bad_pages_and_lengths(fmt, dev):
    """A bad page or a length past the table makes the sequence's live rows NaN and
    touches nothing else; rows behind the live ones stay 0."""
    from naylis_amd.mom_kernels import paged_attention
    c = _case([100, 1900, 50, 64], 4, 2, 64, 16, fmt, dev, N=3, q_lens=[3, 2, 3, 1])
    run = lambda t, n: paged_attention(c["q"], c["cache"], t, n, q_lens=c["q_lens"])  # noqa: E731
    good = run(c["table"], c["lens"])
    table, lens = c["table"].clone(), c["lens"].clone()
    table[1, 30] = len(c["cache"].k)
    table[2, 40:] = 1 << 30
    lens[3] = table.shape[1] * 16 + 1
    got = run(table, lens)
    assert bool(got[1, :2].isnan().all() and got[3, :1].isnan().all())
    assert not bool(got[1, 2:].any()) and not bool(got[3, 1:].any())
    assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    lens[3], lens[0] = 64, -3
    got = run(c["table"], lens)
    assert torch.equal(got[1:], good[1:]) and not bool(got[0].any())


def _e2m1(x):
    """Codes and scale bytes of fp32 rows by the format's definition, on the CPU in fp64."""
    y = x.double().cpu().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1)
    e = (torch.frexp(top)[1] - 3).clamp(min=-126)
    e[top == 0] = -126
    z = y / torch.ldexp(torch.ones_like(top), e)[..., None]
    values = torch.tensor(VALUES, dtype=torch.float64)
    far = (z.abs()[..., None] - values).abs()
    near = far.amin(-1, keepdim=True)
    code = torch.arange(8)
    tie = torch.where(far == near, torch.where(code % 2 == 0, code, code + 8), 99).amin(-1) % 8  # even ones first
    code = (tie | (torch.signbit(z).long() << 3)).flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] | code[..., 1] << 4).to(torch.uint8), (e + 127).to(torch.uint8)


@pytest.mark.parametrize("hd", [64, 128])
def test_e2m1_codes_everywhere(hd, dev):
    """All finite bf16 values beside larger ones of their block: every exponent,
    all ties, values past 6, zeros of both signs, subnormals."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    x = x[x.float().isfinite()]
    g = torch.Generator().manual_seed(hd)
    near = (torch.randint(0, 33, (512, 32), generator=g) / 4.0 * torch.where(torch.rand(512, 32, generator=g) < 0.5, -1.0, 1.0))
    near = (near * 2.0 ** torch.randint(-120, 120, (512, 1), generator=g)).bfloat16()  # multiples of a quarter step
    mixed = x.flatten()[torch.randperm(x.numel(), generator=g)]
    x = torch.cat([x.flatten(), mixed, near.flatten(), torch.zeros(hd).bfloat16()])
    x = torch.cat([x, x.new_zeros((-len(x)) % hd)]).view(-1, 1, hd)
    cache = new_paged_cache(-(-len(x) // 256), 1, 256, hd, dev, fp4=True)
    table = torch.arange(len(cache.k), dtype=torch.int32, device=dev)[None]
    pos = torch.arange(len(x), dtype=torch.int32, device=dev)
    paged_append(cache, x.to(dev), -x.to(dev), table, pos, torch.zeros_like(pos))
    for pages, scale, new in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, -x)):
        codes, e = _e2m1(new.float()[:, 0])
        assert torch.equal(scale.view(-1, hd // 32)[:len(x)].cpu(), e)
        assert torch.equal(pages.view(-1, hd // 2)[:len(x)].cpu(), codes)


def test_e2m1_values(dev):
    """dequantize() and the attention read every code and scale as the format
    defines them, 2^-127 and NaN among the scales."""
    from naylis_amd.mom_kernels import PagedCache, new_paged_cache, paged_attention, paged_gather
    cache = new_paged_cache(16, 1, 16, 64, dev, fp4=True)
    codes = torch.arange(16 * 16 * 32, device=dev).to(torch.uint8).view(16, 1, 16, 32)
    e = torch.arange(256, device=dev).view(16, 1, 16, 1).expand(-1, -1, -1, 2).to(torch.uint8).contiguous()
    cache = PagedCache(codes, codes.flip(-1).contiguous(), e, e)
    values = torch.tensor(VALUES + tuple(-x for x in VALUES), dtype=torch.float64)
    for got, c in zip(cache.dequantize(), cache[:2]):
        c = c.cpu().long()
        want = values[torch.stack([c % 16, c // 16], -1)].flatten(-2).unflatten(-1, (2, 32))
        want = (want * 2.0 ** (e.cpu().double() - 127)[..., None]).flatten(-2)
        want[15, :, 15] = math.nan
        assert torch.equal(got.cpu().double().nan_to_num(7e77), want.float().double().nan_to_num(7e77))
    # one token a sequence: its own value, exact in bf16 (infinite past bf16's largest)
    table = torch.arange(16, dtype=torch.int32, device=dev)[:, None]
    k, v = paged_gather(cache, table, torch.arange(0, 257, 16, dtype=torch.int32, device=dev), 256)
    for got, want in zip((k, v), cache.dequantize()):
        want = want.transpose(1, 2).reshape(256, 1, 64).bfloat16()
        assert torch.equal(got.view(torch.int16)[:255], want.view(torch.int16)[:255]) and bool(got[255].isnan().all())
    q = torch.zeros(16, 1, 64, dtype=torch.bfloat16, device=dev)
    first = paged_attention(q, cache, table, torch.ones(16, dtype=torch.int32, device=dev))
    assert torch.equal(first[1:], v[16::16])
    assert float((first[0].double() - v[0].double()).abs().max()) <= 2.0 ** -126  # a subnormal result


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_e2m1_blocks_that_are_no_numbers(bad, dev):
    """A block with an infinity or a NaN is NaN, in its token and its block alone;
    the sequences that see it in k are NaN, others untouched."""
    from naylis_amd.mom_kernels import paged_append, paged_attention
    c = _case([40, 70], 4, 2, 128, 16, "e2m1", dev)
    good = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    before = [x.clone() for x in c["cache"].dequantize()]
    k = c["k"].clone()
    k[7, 1, 70] = bad
    paged_append(c["cache"], k, c["v"], c["table"], c["pos"], c["rows"])
    after = c["cache"].dequantize()
    page = int(c["table"][0, 0])
    assert bool(after[0][page, 1, 7, 64:96].isnan().all())
    after[0][page, 1, 7, 64:96] = before[0][page, 1, 7, 64:96]
    assert all(torch.equal(a.nan_to_num(7e7), b.nan_to_num(7e7)) for a, b in zip(after, before))
    got = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    assert bool(got[0, 2:].isnan().all()) and torch.equal(got[0, :2], good[0, :2]) and torch.equal(got[1], good[1])


@pytest.mark.parametrize("hd", [64, 128])
def test_e2m1_append_writes_its_rows_alone(hd, dev):
    from naylis_amd.mom_kernels import new_paged_cache, paged_append
    g = torch.Generator(device=dev).manual_seed(hd)
    cache = new_paged_cache(7, 3, 16, hd, dev, fp4=True)
    for t in cache:
        t.copy_(torch.randint(0, 255, t.shape, generator=g, device=dev))
    before = [t.clone() for t in cache]
    T = 40
    k, v = (torch.randn(T, 3, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    table = torch.tensor([[6, 0, 2], [3, 5, 9]], dtype=torch.int32, device=dev)  # page 9 is none
    rows = torch.tensor([i % 2 for i in range(T)], dtype=torch.int32, device=dev)
    pos = torch.tensor([i // 2 for i in range(T)], dtype=torch.int32, device=dev)
    pos[10], pos[11], pos[12], rows[13], rows[14] = -1, 48, 1 << 30, 2, -1
    pos[16], pos[18], pos[17] = 33, 47, 32
    paged_append(cache, k, v, table, pos, rows)
    for new, i in ((k, 0), (v, 1)):
        codes, e = _e2m1(new.float())
        want, scale = before[i].clone(), before[i + 2].clone()
        for t in range(T):
            b, p = int(rows[t]), int(pos[t])
            if not (0 <= b < 2 and 0 <= p < 48) or int(table[b, p // 16]) > 6:
                continue
            want[table[b, p // 16], :, p % 16] = codes[t].to(dev)
            scale[table[b, p // 16], :, p % 16] = e[t].to(dev)
        assert torch.equal(cache[i], want) and torch.equal(cache[i + 2], scale)


@pytest.mark.parametrize("lens", [[1, 40, 33, 300], [3000, 1, 70]])  # tables of one launch, and of two
@pytest.mark.parametrize("size", [2.0 ** 17, 2.0 ** 50, 2.0 ** 60])
def test_e2m1_scores_of_any_size(size, lens, dev):
    """Scores of +-2^30, 2^96 and 2^116: each sequence has a few tokens with the
    highest one, so its result is their mean: weights are 0 or 1, their sum exact,
    and the result is rounded once."""
    from naylis_amd.mom_kernels import paged_append, paged_attention
    c = _case(lens, 4, 2, 128, 16, "e2m1", dev)
    k, q = torch.zeros_like(c["k"]), torch.zeros_like(c["q"])
    q[..., 3] = size
    best = (c["pos"] * 7 + c["rows"]) % 11 == 0
    first = torch.nn.functional.pad(c["lens"].cumsum(0), (1, 0))[:-1].long()
    best[first] = True
    for sign in (-1, 1):
        k[..., 3] = sign * size * torch.where(best, 1.0 if sign > 0 else 0.5, 0.5 if sign > 0 else 1.0)[:, None]
        paged_append(c["cache"], k, c["v"], c["table"], c["pos"], c["rows"])
        got = paged_attention(q, c["cache"], c["table"], c["lens"], scale=0.125).double()
        v = _stored(c, 16)[1]
        for b in range(len(lens)):
            mine = v[(c["rows"] == b) & best]
            want = mine.mean(0).repeat_interleave(2, 0)
            bound = mine.abs().mean(0).repeat_interleave(2, 0) * (2.0 ** -8 + 2.0 ** -20)
            assert bool(((got[b] - want).abs() <= bound).all()), (b, sign)


@pytest.mark.parametrize("fmt", FORMATS)
def test_tokens_streams_and_graph(fmt, dev):
    """Another stream, and two captured graphs of an append and the attention of
    several tokens, replayed on new inputs, lengths and token numbers."""
    from naylis_amd.mom_kernels import paged_append, paged_attention
    c = _case([300, 40, 7], 8, 2, 64, 16, fmt, dev, N=3, q_lens=[3, 1, 2], width=64)
    run = lambda: paged_attention(c["q"], c["cache"], c["table"], c["lens"], q_lens=c["q_lens"])  # noqa: E731
    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    assert torch.equal(got, want)
    k, v, pos, rows = (c[n][290:300].clone() for n in ("k", "v", "pos", "rows"))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            paged_append(c["cache"], k, v, c["table"], pos, rows)
            out = run()
        graphs.append((graph, out))
    g = torch.Generator(device=dev).manual_seed(9)
    for i in range(6):
        c["q"].copy_(torch.randn(c["q"].shape, generator=g, device=dev))
        k.copy_(torch.randn(k.shape, generator=g, device=dev))
        c["lens"].copy_(torch.tensor([300 - 7 * i, 40 - i, 7], dtype=torch.int32))
        c["q_lens"].copy_(torch.tensor([i % 4, 3, (i + 2) % 4], dtype=torch.int32))
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run())


def test_tokens_refusals(dev):
    from naylis_amd.mom_kernels import PagedCache, new_paged_cache, paged_append, paged_attention
    c = _case([20, 30], 4, 2, 64, 16, "e2m1", dev, N=2)
    q, cache, table, lens = c["q"], c["cache"], c["table"], c["lens"]
    k, v, ks, vs = cache
    bad = [(q[:, :0], cache), (q[None], cache), (q[:, :, :3], cache), (q[..., :32], cache), (q.float(), cache),
           (q, PagedCache(k, v, ks, vs.float())), (q, PagedCache(k, v, ks[..., :1].contiguous(), vs)),
           (q, PagedCache(k, v, ks[..., 0].contiguous(), vs[..., 0].contiguous())), (q, PagedCache(k, v)),
           (q, PagedCache(k, v, ks.int(), vs.int())),
           (q, PagedCache(k[..., :16].contiguous(), v[..., :16].contiguous(), ks[..., :1].contiguous(), vs[..., :1].contiguous())),
           (q, PagedCache(k, v, ks.transpose(1, 2), vs))]
    for args in bad:
        with pytest.raises(RuntimeError, match="paged_att"):
            paged_attention(*args, table, lens)
    for q_lens in (lens[:1], lens.float(), lens.cpu(), lens[None]):
        with pytest.raises(RuntimeError, match="q_lens"):
            paged_attention(q, cache, table, lens, q_lens=q_lens)
    with pytest.raises(RuntimeError, match="too many"):
        paged_attention(q.expand(2, 2, 4, 64).repeat(1, 1100, 1, 1), cache, table, lens)
    with pytest.raises(RuntimeError, match="no backward"):
        paged_attention(q.clone().requires_grad_(), cache, table, lens)
    buf = torch.zeros(ks.numel() + 1, dtype=torch.uint8, device=dev)
    for odd in (PagedCache(k, v, buf[1:].view(ks.shape), vs), PagedCache(k, v, ks, buf[1:].view(ks.shape))):
        with pytest.raises(RuntimeError, match="aligned"):
            paged_attention(q, odd, table, lens)
        with pytest.raises(RuntimeError, match="aligned"):
            paged_append(odd, c["k"][:2], c["v"][:2], table, c["pos"][:2])
    with pytest.raises(RuntimeError, match="exclude"):
        new_paged_cache(1, 1, 16, 64, dev, fp8=True, fp4=True)
    assert paged_attention(q[:0], cache, table[:0], lens[:0]).shape == (0, 2, 4, 64)


def test_e2m1_large_cache(dev):
    """Pages whose byte offsets pass 32 bits, and scales past 2^28."""
    from naylis_amd.mom_kernels import PagedCache, paged_append
    pages, Hkv, page, hd = 140000, 8, 64, 128  # 4.6 GB each
    shape = (pages, Hkv, page)
    cache = PagedCache(*(torch.empty(*shape, hd // 2, dtype=torch.uint8, device=dev) for _ in range(2)),
                       *(torch.empty(*shape, hd // 32, dtype=torch.uint8, device=dev) for _ in range(2)))
    g = torch.Generator(device=dev).manual_seed(0)
    n = 150
    k, v = (torch.randn(n, Hkv, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 70]], dtype=torch.int32, device=dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    paged_append(cache, k, v, table, pos, torch.zeros_like(pos))
    ids = table[0].long()
    small = PagedCache(*(t[ids].contiguous() for t in cache))
    c = dict(q=torch.randn(1, 2, 16, hd, generator=g, device=dev).bfloat16(), cache=small, table=torch.arange(3, device=dev)[None],
             rows=torch.zeros_like(pos), pos=pos, lens=torch.tensor([n], dtype=torch.int32, device=dev), q_lens=None)
    want, bound = _attention(c, hd ** -0.5, page)
    from naylis_amd.mom_kernels import paged_attention
    got = paged_attention(c["q"], cache, table, c["lens"])
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("width", [None, 100])  # a table of one launch, and of two
def test_tokens_that_hold_no_numbers(width, fmt, dev):
    """A new token's keys of NaN reach the rows that see it alone; of its values they
    reach the earlier new tokens of its sequence too (a weight of 0 times what it
    stands for), and no other sequence.  A token behind the sequence reaches none."""
    from naylis_amd.mom_kernels import paged_append, paged_attention
    c = _case([70, 45, 33], 4, 2, 64, 16, fmt, dev, N=4, q_lens=[4, 4, 2], width=width)
    run = lambda: paged_attention(c["q"], c["cache"], c["table"], c["lens"], q_lens=c["q_lens"])  # noqa: E731
    good = run()
    last = (c["rows"] == 1) & (c["pos"] == 43)  # seen by the last two of four
    k, v = c["k"].clone(), c["v"].clone()
    k[last] = math.nan
    paged_append(c["cache"], k, c["v"], c["table"], c["pos"], c["rows"])
    got = run()
    assert bool(got[1, 2:].isnan().all()) and torch.equal(got[1, :2], good[1, :2])
    assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    v[last] = math.nan
    paged_append(c["cache"], c["k"], v, c["table"], c["pos"], c["rows"])
    got = run()
    assert bool(got[1, 2:].isnan().all()) and torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    c["lens"][1], c["q_lens"][1] = 43, 2  # the token is behind the sequence now
    got = run()
    assert torch.equal(got[1, :2], good[1, :2])


@pytest.mark.parametrize("fmt", FORMATS)
def test_tokens_one_sequence_among_many(fmt, dev):
    """Sequences that end and begin within a wave's range, 32 rows and two tiles of
    them: the same as each sequence alone, up to where its tokens are cut."""
    from naylis_amd.mom_kernels import paged_attention
    lens = [(i * 37) % 90 + 1 for i in range(150)] + [3000] + [(i * 53) % 70 for i in range(100)]
    for H, N in ((8, 5), (16, 5)):  # 20 rows a key head, 40
        c = _case(lens, H, 2, 128, 16, fmt, dev, N=N, q_lens=[i % (N + 1) for i in range(len(lens))])
        _check(c, 16)


def test_formats_under_trace(dev):
    """A traced attention of several tokens and a traced gather run again on new inputs."""
    from naylis_amd.mom_kernels import paged_attention, paged_gather
    c = _case([70, 45], 4, 2, 64, 16, "e2m1", dev, N=3)
    cu = torch.tensor([0, 70, 115], dtype=torch.int32, device=dev)

    def call(q, lens):
        return paged_attention(q, c["cache"], c["table"], lens, q_lens=lens - 40), *paged_gather(c["cache"], c["table"], cu, 115)
    traced = torch.jit.trace(call, (c["q"], c["lens"]), check_trace=False)
    for q, lens in ((c["q"], c["lens"]), (c["q"].flip(0).contiguous(), c["lens"] - 2)):
        for x, y in zip(traced(q, lens), call(q, lens)):
            assert torch.equal(x, y)


def test_tokens_forward_mode_derivatives_raise(dev):
    import torch.autograd.forward_ad as fwAD
    from naylis_amd.mom_kernels import paged_append_rope, paged_attention, verify_drafts
    c = _case([20, 30], 4, 2, 64, 16, "bf16", dev, N=2)
    x = torch.zeros(2, 3, 50, device=dev)
    with fwAD.dual_level():
        q = fwAD.make_dual(c["q"], torch.ones_like(c["q"]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_attention(q, c["cache"], c["table"], c["lens"])
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_append_rope(c["cache"], q[:, 0], c["k"][:2], c["v"][:2], torch.ones(32, device=dev), c["table"], c["pos"][:2])
        with pytest.raises(RuntimeError, match="forward-mode"):
            verify_drafts(fwAD.make_dual(x, x), torch.zeros(2, 2, dtype=torch.long, device=dev), x[:, :, 0].contiguous())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("B", [1, 2])
def test_tokens_of_the_most_rows(B, fmt, dev):
    """1024 new tokens of 64 heads over 16 key heads, the most rows of a call: q's dense
    stride from sequence to sequence is 2^23."""
    from naylis_amd.mom_kernels import paged_attention
    N, H, Hkv, hd = 1024, 64, 16, 128
    c = _case([1040, 700][:B], H, Hkv, hd, 16, fmt, dev, N=N)
    got = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    k, v = _stored(c, 16)
    at = 0
    for b, n in enumerate(c["lens"].tolist()):
        seen = torch.arange(n, device=dev) <= torch.arange(N, device=dev)[:, None] + n - N  # (N, n)
        for h in range(H):
            x, y = k[at:at + n, h // 4], v[at:at + n, h // 4]
            s = (c["q"][b, :, h].double() @ x.T * hd ** -0.5).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # (rows that see nothing)
            far = (got[b, :, h].double() - p @ y).abs()
            # (as in _attention: the weights and the result are rounded to bf16 once each)
            assert bool((far <= p @ y.abs() * (2.0 ** -7 + 2.0 ** -10) + 1e-30).all())
        at += n


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("Hkv", [1, 4, 8])
def test_tokens_of_a_long_sequence_among_short_ones(Hkv, hd, fmt, dev):
    """A batch whose sequences have few partials on average, and one of which has
    nearly all there are: any number of them is joined."""
    for far in (3001, 6007, 9100):
        lens = [(i * 37) % 90 for i in range(40)] + [far] + [(i * 53) % 70 for i in range(30)]
        c = _case(lens, Hkv, Hkv, hd, 16, fmt, dev, N=3, q_lens=[i % 4 for i in range(len(lens))])
        c["q_lens"][40] = 3
        _check(c, 16)

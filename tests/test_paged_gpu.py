"""paged_append and paged_attention (naylis_mom_paged_*) against fp64 attention
over the gathered tokens: lengths around the 16-token products and the 32 / 64
token steps, empty sequences, long ones among short ones, pages of 16 to 256
tokens, grouped heads up to more than a product holds, bf16 and e4m3."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# lengths, H, Hkv, hd, page, fp8
CASES = [
    ([1], 1, 1, 64, 16, False),
    ([1], 4, 1, 128, 16, True),
    ([0, 1, 15, 16, 17, 31, 32, 33], 4, 2, 64, 16, False),
    ([63, 0, 64, 65, 129, 0], 4, 4, 128, 32, True),
    ([500], 16, 16, 64, 16, False),
    ([5000, 3, 700, 0, 64], 8, 2, 128, 64, False),
    ([9001, 1, 1, 130], 8, 1, 64, 256, True),
    ([40, 300], 34, 2, 128, 128, False),               # 17 query heads a key head
    ([(37 * i) % 400 for i in range(130)], 6, 2, 64, 32, False),
    ([70001], 4, 2, 128, 64, True),
    ([(53 * i) % 900 for i in range(65)], 32, 8, 128, 16, True),
    ([0] * 70 + [600] + [0] * 200 + [(29 * i) % 90 for i in range(100)] + [0], 2, 1, 64, 16, False),
    ([0] * 90 + [5] + [0] * 40, 2, 2, 128, 16, True),
    ([0 if i % 3 else (i * i) % 23 for i in range(4200)] + [530], 2, 1, 64, 16, False),  # chunks of 66 sequences
]


def _case(lens, H, Hkv, hd, page, fp8, dev, seed=0, width=None):
    """A cache whose pages hold NaN (or NaN codes) everywhere but in the live
    rows, which paged_append writes; table entries past the end are -1."""
    from naylis_amd.mom_kernels import PagedCache, paged_append
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
    shape = (pages, Hkv, page, hd)
    if fp8:
        cache = PagedCache(torch.full(shape, 0x7f, dtype=torch.uint8, device=dev),
                           torch.full(shape, 0x7f, dtype=torch.uint8, device=dev),
                           torch.full(shape[:3], math.nan, device=dev), torch.full(shape[:3], math.nan, device=dev))
    else:
        cache = PagedCache(*(torch.full(shape, math.nan, dtype=torch.bfloat16, device=dev) for _ in range(2)))
    T = sum(lens)
    k, v = (torch.randn(T, Hkv, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    q = (torch.randn(len(lens), H, hd, generator=g, device=dev) * 2).bfloat16()
    rows = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(dev, torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev, torch.int32)
    paged_append(cache, k, v, table, pos, rows)
    return dict(q=q, cache=cache, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev), k=k, v=v,
                rows=rows, pos=pos)


def _quantized(x):
    """fp32 rows as the cache holds them: e4m3 codes and scales.  (The divisor is
    a tensor: on the GPU torch multiplies by a number's rounded reciprocal.)"""
    top = x.float().abs().amax(-1)
    s = torch.where(top > 0, top / torch.full_like(top, 448.0), torch.ones_like(top))
    return (x.float() / s[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), s


def _attention(c, scale, fp8):
    """fp64 attention of each sequence over its k, v (as the cache stores them),
    and what bounds the kernel's error: P and the result are rounded to bf16 once
    each, at most 2^-8 relative; exponents and fp32 sums add less than 2^-10."""
    q, k, v = c["q"].double(), c["k"].double(), c["v"].double()
    if fp8:
        k, v = (a.view(torch.float8_e4m3fn).double() * s.double()[..., None] for a, s in
                (_quantized(c["k"]), _quantized(c["v"])))
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    G, at = q.shape[1] // k.shape[1], 0
    for b, n in enumerate(c["lens"].tolist()):
        for h in range(q.shape[1] if n else 0):
            x, y = k[at:at + n, h // G], v[at:at + n, h // G]
            p = torch.softmax(x @ q[b, h] * scale, 0)
            out[b, h], size[b, h] = p @ y, p @ y.abs()
        at += n
    return out, size * (2.0 ** -7 + 2.0 ** -10)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{len(c[0])}-{max(c[0])}-H{c[1]}/{c[2]}x{c[3]}-p{c[4]}-{c[5]}")
def test_paged_matches_fp64(case, dev):
    from naylis_amd.mom_kernels import paged_attention
    c = _case(*case, dev)
    scale = case[3] ** -0.5
    got = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    want, bound = _attention(c, scale, case[5])
    err = (got.double() - want).abs()
    assert bool((err <= bound + 1e-30).all()), float((err / (bound + 1e-30)).max())
    assert torch.equal(got, paged_attention(c["q"], c["cache"], c["table"], c["lens"], scale=scale))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_append_writes_its_rows_alone(fp8, hd, dev):
    """Every row bit for bit, scales and codes as torch's conversion makes them
    (zero rows, tiny and large values among them); padded tokens and tokens
    outside the table or the cache write nothing."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append
    g = torch.Generator(device=dev).manual_seed(hd)
    cache = new_paged_cache(7, 3, 16, hd, dev, fp8=fp8)
    for t in cache:
        if t is not None:
            t.copy_(torch.randint(0, 100, t.shape, generator=g, device=dev))
    before = [None if t is None else t.clone() for t in cache]
    T = 40
    k, v = (torch.randn(T, 3, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    k[0], v[1, 1] = 0, 0
    k[2] *= 1e-38
    k[3] *= 1e30
    v[4, :, 0] = 3e38
    v[5] = torch.linspace(-448, 448, hd, device=dev).bfloat16()
    table = torch.tensor([[6, 0, 2], [3, 5, 9]], dtype=torch.int32, device=dev)  # page 9 is none
    rows = torch.tensor([i % 2 for i in range(T)], dtype=torch.int32, device=dev)
    pos = torch.tensor([i // 2 for i in range(T)], dtype=torch.int32, device=dev)
    pos[10], pos[11], pos[12], rows[13], rows[14] = -1, 48, 1 << 30, 2, -1
    far = pos.long()
    far[10] = (1 << 32) + 3  # beyond int32: out of range, not token 3
    pos[16], pos[18], pos[17] = 33, 47, 32  # row 0's last page; row 1's page 9
    far[16:19] = pos[16:19].long()
    paged_append(cache, k, v, table, far, rows.long())
    for new, pages, old in ((k, cache.k, before[0]), (v, cache.v, before[1])):
        codes, scale = _quantized(new) if fp8 else (new, None)
        want = old.clone()
        ws = before[2 if new is k else 3]
        ws = None if ws is None else ws.clone()
        for t in range(T):
            b, p = int(rows[t]), int(pos[t])
            if not (0 <= b < 2 and 0 <= p < 48) or int(table[b, p // 16]) > 6:
                continue
            want[table[b, p // 16], :, p % 16] = codes[t]
            if fp8:
                ws[table[b, p // 16], :, p % 16] = scale[t]
        assert torch.equal(pages.view(torch.uint8 if fp8 else torch.int16), want.view(torch.uint8 if fp8 else torch.int16))
        if fp8:
            assert torch.equal(cache.k_scale if new is k else cache.v_scale, ws)


def test_append_codes_match_torch_everywhere(dev):
    """All bf16 values of a row's range, as codes: the conversion rounds to
    nearest even at every step of the format, subnormals and signed zeros too."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append
    bits = torch.arange(0, 1 << 16, device=dev).to(torch.int32)
    x = bits.to(torch.int16).view(torch.bfloat16)
    x = x[(x.float().abs() <= 448)]
    x = torch.cat([x, x.new_full(((-len(x)) % 63,), 1.0)]).view(-1, 63)
    x = torch.cat([x, x.new_full((len(x), 1), 448.0)], 1).view(-1, 1, 64)  # scale 1
    cache = new_paged_cache(-(-len(x) // 256), 1, 256, 64, dev, fp8=True)
    table = torch.arange(len(cache.k), dtype=torch.int32, device=dev)[None]
    pos = torch.arange(len(x), dtype=torch.int32, device=dev)
    paged_append(cache, x, x, table, pos, torch.zeros_like(pos))
    want = x.float().to(torch.float8_e4m3fn).view(torch.uint8)[:, 0]
    assert torch.equal(cache.k.view(-1, 64)[:len(x)], want) and torch.equal(cache.v.view(-1, 64)[:len(x)], want)


def test_bad_pages_and_lengths(dev):
    """A page outside the cache, or a length past the table's row, makes that
    sequence NaN and touches no other; entries past the end do not count."""
    from naylis_amd.mom_kernels import paged_attention
    for fp8 in (False, True):
        c = _case([100, 900, 50, 64], 4, 2, 64, 16, fp8, dev)
        good = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
        table, lens = c["table"].clone(), c["lens"].clone()
        table[1, 30] = len(c["cache"].k)
        table[2, 40:] = 1 << 30
        lens[3] = table.shape[1] * 16 + 1
        got = paged_attention(c["q"], c["cache"], table, lens)
        assert bool(got[1].isnan().all() and got[3].isnan().all())
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
        table[1, 30] = -7
        lens[3], lens[0] = 64, -3
        got = paged_attention(c["q"], c["cache"], table, lens)
        assert bool(got[1].isnan().all()) and torch.equal(got[2:], good[2:]) and bool((got[0] == 0).all())


def test_paged_result_depends_on_its_sequence_alone(dev):
    """The same sequence alone and in a batch: equal up to where its tokens are
    cut (fp32 joins, one bf16 rounding each)."""
    from naylis_amd.mom_kernels import paged_attention
    c = _case([3000, 10, 4000], 8, 2, 128, 32, False, dev)
    both = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    one = paged_attention(c["q"][:1], c["cache"], c["table"][:1], c["lens"][:1])
    # both sides: P rounded at another reference, the result rounded: 2^-7 of sum p |v| each
    want, bound = _attention(c, 128 ** -0.5, False)
    assert bool(((one[0].double() - both[0].double()).abs() <= 2 * bound[0]).all())


def test_paged_large_cache(dev):
    """Pages whose byte offsets pass 32 bits."""
    from naylis_amd.mom_kernels import PagedCache, paged_append, paged_attention
    pages, Hkv, page, hd = 40000, 8, 64, 128  # 5.2 GB each
    cache = PagedCache(*(torch.empty(pages, Hkv, page, hd, dtype=torch.bfloat16, device=dev) for _ in range(2)))
    g = torch.Generator(device=dev).manual_seed(0)
    n = 150
    k, v = (torch.randn(n, Hkv, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    table = torch.tensor([[39999, 3, 35000]], dtype=torch.int32, device=dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    paged_append(cache, k, v, table, pos, torch.zeros_like(pos))
    assert torch.equal(cache.k[39999, :, :].transpose(0, 1), k[:64])
    q = torch.randn(1, 16, hd, generator=g, device=dev).bfloat16()
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    c = dict(q=q, k=k, v=v, lens=lens)
    want, bound = _attention(c, hd ** -0.5, False)
    got = paged_attention(q, cache, table, lens)
    assert bool(((got.double() - want).abs() <= bound).all())


def test_paged_views_streams_and_graph(dev):
    """q as a slice of a projection, int64 tables, another stream, and a captured
    append + attention replayed on new inputs and lengths with eager calls (and
    a second captured graph) between."""
    from naylis_amd.mom_kernels import PagedCache, paged_append, paged_attention
    c = _case([300, 40, 7], 8, 2, 64, 16, False, dev, width=32)
    want = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    wide = torch.cat([c["q"].flatten(1), c["q"].flatten(1)], 1)
    assert torch.equal(paged_attention(wide[:, 512:].view(3, 8, 64), c["cache"], c["table"].long(), c["lens"].long()), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged_attention(c["q"], c["cache"], c["table"], c["lens"])
    s.synchronize()
    assert torch.equal(got, want)

    # one free page for each sequence's next token where its pages are full
    table = c["table"].clone()
    cache = PagedCache(*(torch.cat([t, t.new_full((3, *t.shape[1:]), math.nan)]) for t in c["cache"][:2]))
    for b, n in enumerate((300, 40, 7)):
        if n % 16 == 0:
            table[b, n // 16] = len(cache.k) - 1 - b
    held = dict(q=c["q"].clone(), k=torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev),
                v=torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev), pos=c["lens"].clone(), lens=c["lens"] + 1)
    graphs = []
    paged_attention(held["q"], cache, table, c["lens"])
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            paged_append(cache, held["k"], held["v"], table, held["pos"])
            out = paged_attention(held["q"], cache, table, held["lens"])
        graphs.append((graph, out))
    g = torch.Generator(device=dev).manual_seed(9)
    for i in range(4):
        for n in ("q", "k", "v"):
            held[n].copy_(torch.randn(held[n].shape, generator=g, device=dev))
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        eager = paged_attention(held["q"], cache, table, held["lens"])
        assert torch.equal(out, eager)
        for b, n in enumerate((300, 40, 7)):
            assert torch.equal(cache.k[table[b, n // 16], :, n % 16], held["k"][b])


def test_paged_single_sequence_of_odd_rows(dev):
    """One sequence's q, k, v out of a tensor whose rows are no whole 16-byte pieces."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append, paged_attention
    x = torch.randn(2, 389, generator=torch.Generator(device=dev).manual_seed(4), device=dev).bfloat16()
    q, k, v = (torch.as_strided(x, (1, 2, 64), (389, 64, 1), 128 * i) for i in range(3))
    cache = new_paged_cache(1, 2, 16, 64, dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    paged_append(cache, k, v, table, torch.zeros(1, dtype=torch.int32, device=dev))
    assert torch.equal(cache.k[0, :, 0], k[0]) and torch.equal(cache.v[0, :, 0], v[0])
    assert torch.equal(paged_attention(q, cache, table, torch.ones(1, dtype=torch.int32, device=dev)), v)


def test_paged_append_marks_the_cache_written(dev):
    """A graph that saved the cache notices the write."""
    from naylis_amd.mom_kernels import paged_append
    c = _case([20], 2, 1, 64, 16, False, dev)
    w = torch.ones((), device=dev, requires_grad=True)
    y = (c["cache"].k[:1].nan_to_num() * w).sum() + (c["cache"].v * w).sum()
    paged_append(c["cache"], c["k"][:1], c["v"][:1], c["table"], c["pos"][:1])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_paged_refusals(dev):
    from naylis_amd.mom_kernels import PagedCache, paged_append, paged_attention
    c = _case([20, 3], 4, 2, 64, 16, False, dev)
    f = _case([20, 3], 4, 2, 64, 16, True, dev)
    q, cache, table, lens = c["q"], c["cache"], c["table"], c["lens"]
    t = lambda x: x.transpose(2, 3)  # noqa: E731
    bad = [(q.float(), cache, table, lens), (q[:, :3], cache, table, lens), (q, cache, table[:1], lens),
           (q, cache, table, lens[:1]), (q, cache, table.cpu(), lens), (q, cache, table, lens.float()),
           (q[..., :32], cache, table, lens), (q, PagedCache(cache.k, cache.v.float()), table, lens),
           (q, PagedCache(t(cache.k), t(cache.v)), table, lens), (q, PagedCache(*f["cache"][:2]), table, lens),
           (q, PagedCache(*cache[:2], *f["cache"][2:]), table, lens), (q, cache, table[:, :0], lens),
           (q, PagedCache(cache.k[:, :, :8].contiguous(), cache.v[:, :, :8].contiguous()), table, lens),
           (q, PagedCache(*f["cache"][:2], f["cache"].k_scale[:, :1], f["cache"].v_scale), table, lens)]
    for args in bad:
        with pytest.raises(RuntimeError, match="paged_att"):
            paged_attention(*args)
    with pytest.raises(RuntimeError, match="scale"):
        paged_attention(q, cache, table, lens, scale=0.0)
    with pytest.raises(RuntimeError, match="no backward"):
        paged_attention(q.clone().requires_grad_(), cache, table, lens)
    with pytest.raises(RuntimeError, match="no backward"):
        paged_append(cache, c["k"][:2].clone().requires_grad_(), c["v"][:2], table, c["pos"][:2])
    k, v, pos = c["k"][:2], c["v"][:2], c["pos"][:2]
    bad = [(cache, k.float(), v.float(), table, pos), (cache, k, v[:1], table, pos), (cache, k[:, :1], v[:, :1], table, pos),
           (cache, k, v, table, pos[:1]), (cache, k, v, table, pos, pos[:1]), (cache, k, v, table[0], pos),
           (cache, k, v, table, pos.float()), (cache, c["k"][:3], c["v"][:3], table, c["pos"][:3]),
           (cache, k, v, table.cpu(), pos)]
    for args in bad:
        with pytest.raises(RuntimeError, match="paged_append"):
            paged_append(*args)
    assert paged_attention(q[:0], cache, table[:0], lens[:0]).shape == (0, 4, 64)
    paged_append(cache, k[:0], v[:0], table, pos[:0])


def test_paged_scales_out_of_line_are_refused(dev):
    """Dense scales that begin off a 16-byte boundary of a larger buffer."""
    from naylis_amd.mom_kernels import PagedCache, paged_append, paged_attention
    c = _case([20, 3], 4, 2, 64, 16, True, dev)
    k, v, ks, vs = c["cache"]
    for off in (1, 2, 3):
        buf = torch.ones(ks.numel() + off, device=dev)
        odd = buf[off:].view(ks.shape)
        assert odd.is_contiguous()
        for cache in (PagedCache(k, v, odd, vs), PagedCache(k, v, ks, odd)):
            with pytest.raises(RuntimeError, match="paged_attention.*aligned"):
                paged_attention(c["q"], cache, c["table"], c["lens"])
            with pytest.raises(RuntimeError, match="paged_append.*aligned"):
                paged_append(cache, c["k"][:2], c["v"][:2], c["table"], c["pos"][:2])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[1, 40, 33, 300], [3000, 1, 70]])  # tables of one launch, and of two
@pytest.mark.parametrize("size", [2.0 ** 17, 2.0 ** 50, 2.0 ** 60])
def test_paged_scores_of_any_size(size, lens, hd, fp8, dev):
    """Scores of +-2^30, 2^96 and 2^116: each sequence has a few tokens with the
    highest one, so its result is their mean; once with all scores negative, once
    positive.  Weights are 0 or 1, their sum exact, e4m3 values times their scale
    rounded once to bf16, and the result once: 2^-8 each of the values."""
    from naylis_amd.mom_kernels import PagedCache, paged_append, paged_attention
    c = _case(lens, 4, 2, hd, 16, fp8, dev)
    k, q = torch.zeros_like(c["k"]), torch.zeros_like(c["q"])
    q[..., 3] = size
    best = (c["pos"] * 7 + c["rows"]) % 11 == 0
    first = torch.nn.functional.pad(c["lens"].cumsum(0), (1, 0))[:-1].long()
    best[first] = True
    for sign in (-1, 1):
        k[..., 3] = sign * size * torch.where(best, 1.0 if sign > 0 else 0.5, 0.5 if sign > 0 else 1.0)[:, None]
        paged_append(c["cache"], k, c["v"], c["table"], c["pos"], c["rows"])
        got = paged_attention(q, c["cache"], c["table"], c["lens"], scale=0.125).double()
        _, v = PagedCache(*c["cache"]).dequantize()
        page, off = c["table"][c["rows"].long(), c["pos"].long() // 16].long(), c["pos"].long() % 16
        v = v.double()[page, :, off]
        for b in range(len(lens)):
            mine = v[(c["rows"] == b) & best]
            want = mine.mean(0).repeat_interleave(2, 0)
            bound = mine.abs().mean(0).repeat_interleave(2, 0) * (2.0 ** -7 + 2.0 ** -20)
            assert bool(((got[b] - want).abs() <= bound).all()), (b, sign)

"""paged_append_rope and paged_gather against fp64 statements: positions from 0
to the far end, whole and partial rotations, the three kinds of pages, tokens
that are left out, sequences back dense."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FORMATS = ("bf16", "e4m3", "e2m1")


def _freq(half, dev, base=10000.0):
    return (base ** (-torch.arange(half, device=dev).double() / half)).float()


def _turned(x, pos, freq, scaling=1.0):
    """fp64 rotation, and what bounds an fp32 one: cos and sin (times the scaling)
    are rounded twice at most, each product and the sum once: 2^-24 of a product's
    size each, less than 2^-22 of the pair's sizes in all."""
    half, x = freq.numel(), x.double()
    z = torch.complex(x[..., :half], x[..., half:2 * half])
    angle = pos.double()[:, None] * freq.double()
    y = z * torch.polar(torch.full_like(angle, scaling), angle)[:, None]
    size = (x[..., :half].abs() + x[..., half:2 * half].abs()) * abs(scaling)
    rest = x[..., 2 * half:]
    return (torch.cat([y.real, y.imag, rest], -1),
            torch.cat([size, size, torch.zeros_like(rest)], -1) * 2.0 ** -22)


def _new(T, H, Hkv, hd, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + T + H + hd)
    return [torch.randn(T, h, hd, generator=g, device=dev).bfloat16() for h in (H, Hkv, Hkv)]


def _scattered(lens, page, dev, seed=0):
    """A table of scattered pages, the tokens' rows and positions, the number of pages."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(need) + 2, generator=g)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    rows = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(dev, torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev, torch.int32)
    return table.to(dev), rows, pos, len(ids)


@pytest.mark.parametrize("hd,half", [(64, 32), (64, 16), (64, 8), (64, 24), (128, 64), (128, 32), (128, 40), (128, 8)])
def test_rotation_matches_fp64(hd, half, dev):
    """Queries at positions up to 2^31 - 1 and below 0, and keys where they fit."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append_rope
    T, H, Hkv = 37, 5, 3
    q, k, v = _new(T, H, Hkv, hd, dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    pos[20:30] = torch.tensor([131071, 131070, 1 << 20, (1 << 24) + 1, (1 << 30) - 7, 2 ** 31 - 1, -1, -5000, 99999, 65537])
    freq = _freq(half, dev)
    cache = new_paged_cache(3, Hkv, 16, hd, dev)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    for scaling in (1.0, 0.7):
        for t in cache[:2]:
            t.zero_()
        got = paged_append_rope(cache, q, k, v, freq, table, pos, torch.zeros_like(pos), attention_scaling=scaling)
        want, near = _turned(q, pos, freq, scaling)
        assert bool(((got.double() - want).abs() <= near + want.abs() * 2.0 ** -8).all())
        want, near = _turned(k, pos, freq, scaling)
        at = [i for i in range(T) if 0 <= int(pos[i]) < 48]
        p = pos[at].long()
        held = cache.k[table[0, p // 16].long(), :, p % 16].double()
        assert bool(((held - want[at]).abs() <= (near + want.abs() * 2.0 ** -8)[at]).all())
        assert torch.equal(cache.v[table[0, p // 16].long(), :, p % 16], v[at])
        free = torch.ones(3, 16, dtype=torch.bool, device=dev)
        free[table[0, p // 16].long(), p % 16] = False
        assert not bool(cache.k.transpose(1, 2)[free].any()) and not bool(cache.v.transpose(1, 2)[free].any())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd,half", [(64, 32), (128, 64), (128, 24)])
def test_rotated_keys_as_codes(hd, half, fmt, dev):
    """Codes of the rotated rows before any other rounding: each value within half
    a step of its own (e4m3: 2^-4 of it or 2^-10 of the scale; e2m1: a quarter of
    the scale below 2, a half below 4, one up to 6, two where 6 stands for up to 8)."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append, paged_append_rope
    lens = [300, 17, 1]
    table, rows, pos, pages = _scattered(lens, 32, dev)
    _, k, v = _new(sum(lens), 1, 2, hd, dev)
    freq = _freq(half, dev)
    make = lambda: new_paged_cache(pages, 2, 32, hd, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1")  # noqa: E731
    cache, plain = make(), make()
    assert paged_append_rope(cache, None, k, v, freq, table, pos, rows) is None
    paged_append(plain, k, v, table, pos, rows)
    assert torch.equal(cache.v, plain.v) and torch.equal(cache.v_scale, plain.v_scale)
    at, off = table[rows.long(), pos.long() // 32].long(), pos.long() % 32
    got = cache.dequantize()[0][at, :, off].double()
    want, near = _turned(k, pos, freq)
    if fmt == "e4m3":
        s = cache.k_scale[at, :, off].double()[..., None]
        top = want.abs().amax(-1, keepdim=True)
        assert bool(((s - top / 448).abs() <= near.amax(-1, keepdim=True) / 448 + s * 2.0 ** -23).all())
        step = torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10)
        step += s * 2.0 ** -16  # the scale's own rounding moves 448 by an ulp or two
    else:
        e = cache.k_scale[at, :, off].double()
        top = want.unflatten(-1, (-1, 32)).abs().amax(-1)
        exact = torch.floor(torch.log2(top)) + 125
        clear = (torch.log2(top) - torch.round(torch.log2(top))).abs() > 2.0 ** -18  # away from a power of two
        assert torch.equal(e[clear], exact[clear]) and bool(((e - exact).abs() <= 1).all())
        s = (2.0 ** (e - 127)).repeat_interleave(32, -1)
        a = want.abs() / s
        step = s * torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, torch.where(a <= 6, 1.0, 2.0))) + s * 2.0 ** -16
    assert bool(((got - want).abs() <= step + near).all())


def test_rotation_is_the_decoders(dev):
    """The same rows through ``rope`` with transformers' cosines: the two differ by
    the roundings that it keeps (cos, sin, two products, a sum: 2^-8 each of the
    pair's sizes) and this one's."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append_rope
    from naylis_amd.mom_kernels.hip_rope import rope
    T, H, hd = 200, 4, 64
    q, k, v = _new(T, H, H, hd, dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    freq = _freq(hd // 2, dev)
    angle = torch.cat([pos.float()[:, None] * freq] * 2, -1)[None]
    a, b = rope(q[None], k[None], angle.cos().bfloat16(), angle.sin().bfloat16())
    cache = new_paged_cache(13, H, 16, hd, dev)
    table = torch.arange(13, dtype=torch.int32, device=dev)[None]
    got = paged_append_rope(cache, q, k, v, freq, table, pos, torch.zeros_like(pos))
    held = cache.k.transpose(1, 2).reshape(-1, H, hd)[:T]
    for mine, other, x in ((got, a[0], q), (held, b[0], k)):
        size = (x.double().abs() + x.double().roll(hd // 2, -1).abs()) * 2.0 ** -8
        assert bool(((mine.double() - other.double()).abs() <= 4 * size).all())


def test_append_rope_leaves_tokens_out(dev):
    """Padding, rows and pages that are none: nothing else is written, and every
    query is rotated to its position all the same."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append_rope
    for fmt in FORMATS:
        cache = new_paged_cache(7, 2, 16, 64, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1")
        q, k, v = _new(6, 4, 2, 64, dev)
        table = torch.tensor([[6, 0, 2], [3, 5, 9]], dtype=torch.int32, device=dev)  # page 9 is none
        pos = torch.tensor([-1, 48, 40, 3, 3, 2], dtype=torch.int32, device=dev)
        rows = torch.tensor([0, 0, 1, 2, -1, 1], dtype=torch.int32, device=dev)
        before = [None if t is None else t.clone() for t in cache]
        got = paged_append_rope(cache, q, k, v, _freq(32, dev), table, pos, rows)
        for t, old in zip(cache, before):
            if t is not None:
                same = t == old
                same[3, :, 2] = True  # the last token's place
                assert bool(same.all())
        assert bool(cache.k[3, :, 2].any())
        want, near = _turned(q, pos, _freq(32, dev))
        assert bool(((got.double() - want).abs() <= near + want.abs() * 2.0 ** -8).all())


def test_append_rope_views_streams_and_graph(dev):
    """Operands as slices of one projection, rows of their own number without
    ``rows``, another stream, and a captured call replayed at new positions."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append_rope
    T, H, Hkv, hd = 4, 6, 2, 128
    x = torch.randn(T, H + 2 * Hkv, hd, generator=torch.Generator(device=dev).manual_seed(1), device=dev).bfloat16()
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    freq = _freq(64, dev)
    table = torch.arange(8, dtype=torch.int32, device=dev).view(4, 2)
    pos = torch.tensor([0, 31, 16, 5], dtype=torch.int32, device=dev)
    caches = [new_paged_cache(8, Hkv, 16, hd, dev) for _ in range(4)]
    want = paged_append_rope(caches[0], q.contiguous(), k.contiguous(), v.contiguous(), freq, table, pos)
    assert torch.equal(paged_append_rope(caches[1], q, k, v, freq, table.long(), pos.long()), want)
    odd = torch.cat([x[..., :1], x], -1)[..., 1:]
    assert torch.equal(paged_append_rope(caches[2], odd[:, :H], odd[:, H:H + Hkv], odd[:, H + Hkv:], freq, table, pos), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged_append_rope(caches[3], q, k, v, freq, table, pos)
    s.synchronize()
    assert torch.equal(got, want)
    for c in caches[1:]:
        assert torch.equal(c.k, caches[0].k) and torch.equal(c.v, caches[0].v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = paged_append_rope(caches[1], q, k, v, freq, table, pos)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(2 + i), device=dev))
        pos.copy_(torch.tensor([i, 30 - i, 17 + i, 8], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_append_rope(caches[2], q, k, v, freq, table, pos))
        at, off = table[torch.arange(4, device=dev), pos.long() // 16].long(), pos.long() % 16
        assert torch.equal(caches[1].k[at, :, off], caches[2].k[at, :, off])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,Hkv,hd,page", [([1], 1, 64, 16), ([0, 40, 0, 0, 17, 16, 300, 0], 3, 128, 16),
                                              ([2000, 1, 999], 2, 64, 64), ([(31 * i) % 57 for i in range(300)], 1, 128, 32)])
def test_gather_gives_the_cache_back(lens, Hkv, hd, page, fmt, dev):
    """Every row bit for bit: bf16 and e2m1 exact, e4m3 code times scale rounded
    once; rows before the first offset and behind the last are 0."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append, paged_gather
    table, rows, pos, pages = _scattered(lens, page, dev, seed=len(lens))
    _, k, v = _new(sum(lens), 1, Hkv, hd, dev)
    cache = new_paged_cache(pages, Hkv, page, hd, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1")
    paged_append(cache, k, v, table, pos, rows)
    at, off = table[rows.long(), pos.long() // page].long(), pos.long() % page
    want = [x[at, :, off].bfloat16() for x in cache.dequantize()]
    for lead, tail in ((0, 0), (5, 9)):
        cu = torch.tensor([lead] + (lead + torch.tensor(lens).cumsum(0)).tolist(), dtype=torch.int32, device=dev)
        T = lead + sum(lens) + tail
        for x, y in zip(paged_gather(cache, table, cu, T), want):
            assert x.shape == (T, Hkv, hd) and torch.equal(x[lead:lead + sum(lens)], y)
            assert not bool(x[:lead].any()) and not bool(x[T - tail:].any())
        short = max(sum(lens) - 7, 0)
        for x, y in zip(paged_gather(cache, table, cu - lead, short), want):
            assert torch.equal(x, y[:short])
    assert torch.equal(paged_gather(cache, table, (cu - lead).long(), sum(lens))[0], want[0])


@pytest.mark.parametrize("fmt", FORMATS)
def test_gather_bad_pages(fmt, dev):
    """Pages outside the cache and tokens past the table's row are NaN, alone."""
    from naylis_amd.mom_kernels import new_paged_cache, paged_append, paged_gather
    table, rows, pos, pages = _scattered([40, 20], 16, dev)
    _, k, v = _new(60, 1, 2, 64, dev)
    cache = new_paged_cache(pages, 2, 16, 64, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1")
    paged_append(cache, k, v, table, pos, rows)
    cu = torch.tensor([0, 50, 70], dtype=torch.int32, device=dev)  # ten tokens past the first row's 48
    bad = table.clone()
    bad[0, 1], bad[1, 0] = pages, -9
    good, got = paged_gather(cache, table, torch.tensor([0, 40, 60], dtype=torch.int32, device=dev), 60), paged_gather(cache, bad, cu, 70)
    for x, y in zip(got, good):
        assert bool(x[16:32].isnan().all() and x[48:66].isnan().all())
        assert torch.equal(x[:16], y[:16]) and torch.equal(x[32:40], y[32:40]) and torch.equal(x[66:], y[56:])
    assert paged_gather(cache, bad, cu, 0)[0].shape == (0, 2, 64)


def test_chunk_in_a_graph(dev):
    """A chunk's append, its gather and the packed attention over it in one captured
    graph, replayed with new tokens, places and lengths."""
    from naylis_amd.mom_kernels import new_paged_cache, packed_attention, paged_append_rope, paged_gather
    B, W, T, Hkv, hd = 3, 6, 40, 2, 64
    caches = [new_paged_cache(B * W, Hkv, 16, hd, dev, fp4=True) for _ in range(2)]
    table = torch.randperm(B * W, generator=torch.Generator().manual_seed(0)).view(B, W).int().to(dev)
    q, k, v = _new(T, 4, Hkv, hd, dev)
    freq = _freq(32, dev)
    rows, pos = torch.zeros(T, dtype=torch.int32, device=dev), torch.arange(T, dtype=torch.int32, device=dev)
    cu_q, cu_k = (torch.tensor([0, T, T, T], dtype=torch.int32, device=dev) for _ in range(2))

    def chunk(cache):
        r = paged_append_rope(cache, q, k, v, freq, table, pos, rows)
        kd, vd = paged_gather(cache, table, cu_k, 150)
        return packed_attention(r, kd, vd, cu_q, cu_k)
    chunk(caches[0])
    for t in caches[0]:
        t.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = chunk(caches[0])
    start = [0, 0, 0]
    for i in range(5):
        for t, new in zip((q, k, v), _new(T, 4, Hkv, hd, dev, seed=i + 1)):
            t.copy_(new)
        add = [(10, 15, 15), (1, 38, 1), (20, 0, 20), (13, 13, 14), (0, 1, 39)][i]
        rows.copy_(torch.repeat_interleave(torch.arange(B), torch.tensor(add)))
        pos.copy_(torch.cat([torch.arange(a, a + n) for a, n in zip(start, add)]))
        start = [(a + n) % 50 for a, n in zip(start, add)]
        ends = [int(pos[rows == b].max()) + 1 if n else 0 for b, n in enumerate(add)]
        cu_q.copy_(torch.tensor([0, *torch.tensor(add).cumsum(0).tolist()]))
        cu_k.copy_(torch.tensor([0, *torch.tensor(ends).cumsum(0).tolist()]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, chunk(caches[1]))
        assert all(torch.equal(x, y) for x, y in zip(*(c[:2] for c in caches)))


def test_chunk_refusals(dev):
    from naylis_amd.mom_kernels import PagedCache, new_paged_cache, paged_append_rope, paged_gather
    cache = new_paged_cache(4, 2, 16, 64, dev)
    q, k, v = _new(3, 4, 2, 64, dev)
    table = torch.zeros(3, 1, dtype=torch.int32, device=dev)
    pos, freq = torch.zeros(3, dtype=torch.int32, device=dev), _freq(32, dev)
    call = lambda cache=cache, q=q, k=k, v=v, freq=freq, table=table, pos=pos, **kw: paged_append_rope(  # noqa: E731
        cache, q, k, v, freq, table, pos, **kw)
    for kw in (dict(q=q[:2]), dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[:, :0]), dict(q=q[0]), dict(k=k.float()), dict(v=v[:2]),
               dict(k=k[:, :1], v=v[:, :1]), dict(freq=freq.double()), dict(freq=freq[None]), dict(freq=freq.cpu()), dict(freq=_freq(40, dev)),
               dict(freq=freq[:12]), dict(freq=freq[:0]), dict(pos=pos[:2]), dict(pos=pos.float()), dict(table=table[0]),
               dict(table=table[:2]), dict(rows=pos[:1]), dict(attention_scaling=math.inf), dict(attention_scaling=math.nan),
               dict(cache=PagedCache(cache.k, cache.v.float())), dict(q=q.cpu())):
        with pytest.raises(RuntimeError, match="paged_append_rope"):
            call(**kw)
    for kw in (dict(q=q.clone().requires_grad_()), dict(k=k.clone().requires_grad_()), dict(freq=freq.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no backward"):
            call(**kw)
    assert call(q=q[:0], k=k[:0], v=v[:0], pos=pos[:0]).shape == (0, 4, 64)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
    for args in ((cache, table[0], cu, 3), (cache, table, cu[:3], 3), (cache, table, cu.float(), 3), (cache, table, cu, -1),
                 (cache, table.cpu(), cu, 3), (PagedCache(cache.k, cache.v.float()), table, cu, 3), (cache, table[:0], cu[:1], 3)):
        with pytest.raises(RuntimeError, match="paged_gather"):
            paged_gather(*args)


def test_append_rope_marks_the_cache_written(dev):
    from naylis_amd.mom_kernels import new_paged_cache, paged_append_rope
    cache = new_paged_cache(1, 2, 16, 64, dev)
    q, k, v = _new(1, 4, 2, 64, dev)
    w = torch.ones((), device=dev, requires_grad=True)
    y = (cache.k * w).sum()
    zero = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    paged_append_rope(cache, q, k, v, _freq(32, dev), zero, zero[0])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()

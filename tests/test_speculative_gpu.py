"""A speculative serving loop as a program runs it: a prompt rotated into the
cache and read back dense for the packed pass, then steps that append the last
token with its drafts, read the cache for all of them and verify them; hidden
states against the packed pass over the whole sequences, tokens against the
logits' own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, HKV, HD, V, LAYERS, N, PAGE = 256, 4, 2, 64, 1000, 2, 3, 16
# a layer's attention is within 2^-7 of itself on either side, each bf16
# projection and sum a rounding more, over two layers; e4m3 rows are off by at
# most 2^-4 of themselves and e2m1 rows by a quarter, keys and values alike
FAR = {"bf16": 2.0 ** -5, "e4m3": 2.0 ** -2, "e2m1": 2.0 ** -1}


def _weights(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: (torch.randn(*s, generator=g, device=dev) * s[0] ** -0.5).bfloat16()  # noqa: E731
    return dict(embed=(torch.randn(V, D, generator=g, device=dev)).bfloat16(),
                layers=[dict(q=r(D, H * HD), k=r(D, HKV * HD), v=r(D, HKV * HD), o=r(H * HD, D)) for _ in range(LAYERS)],
                head=r(D, V), freq=(10000.0 ** (-torch.arange(HD // 2, device=dev).double() / (HD // 2))).float())


def _layer(x, w, attend):
    h = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5)
    h = h.bfloat16()
    q, k, v = ((h @ w[n]).view(len(x), -1, HD) for n in "qkv")
    return x + attend(q, k, v).reshape(len(x), -1) @ w["o"]


def _turned(x, pos, freq):
    angle = pos.double()[:, None, None] * freq.double()
    c, s = angle.cos().float(), angle.sin().float()
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16()


def _places(lens, dev):
    rows = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(dev, torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev, torch.int32)
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev), rows, pos


def _whole(w, tokens, lens, dev):
    """Hidden states of whole sequences, packed, without a cache."""
    from naylis_amd import mom_kernels as mk
    cu, rows, pos = _places(lens, dev)
    x = w["embed"][tokens[rows.long(), pos.long()]]
    for lw in w["layers"]:
        x = _layer(x, lw, lambda q, k, v: mk.packed_attention(_turned(q, pos, w["freq"]), _turned(k, pos, w["freq"]), v, cu))
    return x, cu.tolist()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "e2m1"])
def test_speculative_steps_match_the_whole(fmt, dev):
    from naylis_amd import mom_kernels as mk
    w = _weights(dev)
    g = torch.Generator(device=dev).manual_seed(1)
    prompts, steps = [37, 1, 130, 64], 6
    B = len(prompts)
    width = -(-(max(prompts) + (steps + 1) * (N + 1)) // PAGE)
    tokens = torch.randint(0, V, (B, width * PAGE), generator=g, device=dev)
    table = torch.randperm(B * width + 1, generator=g, device=dev)[:B * width].view(B, width).int()
    caches = [mk.new_paged_cache(B * width + 1, HKV, PAGE, HD, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1") for _ in range(LAYERS)]

    def near(x, want):
        far = float((x.float() - want.float()).norm() / want.float().norm())
        assert far < FAR[fmt], far

    # the prompts, but for the last tokens, which the first step takes
    lens = [n - 1 for n in prompts]
    cu, rows, pos = _places(lens, dev)
    x = w["embed"][tokens[rows.long(), pos.long()]]
    for c, lw in zip(caches, w["layers"]):
        def attend(q, k, v):
            q = mk.paged_append_rope(c, q, k, v, w["freq"], table, pos, rows)
            k, v = mk.paged_gather(c, table, cu, len(q))
            return mk.packed_attention(q, k, v, cu)
        x = _layer(x, lw, attend)
    near(x, _whole(w, tokens, lens, dev)[0])

    row = torch.arange(B, device=dev)

    def step(last, drafts, live):
        """Hidden states (B, N + 1, D) of the last tokens and their drafts, at last[b] .."""
        new = torch.cat([tokens[row, last][:, None], drafts], 1)
        at = last[:, None] + torch.arange(N + 1, device=dev)
        at = torch.where(at <= (last + live)[:, None], at, -1)  # drafts that are none are padding
        x = w["embed"][new.flatten()]
        for c, lw in zip(caches, w["layers"]):
            def attend(q, k, v):
                q = mk.paged_append_rope(c, q, k, v, w["freq"], table, at.flatten().int(), row.repeat_interleave(N + 1).int())
                return mk.paged_attention(q.view(B, N + 1, H, HD), c, table, last + live + 1, q_lens=live + 1)
            x = _layer(x, lw, attend)
        return x.view(B, N + 1, D)

    last = torch.tensor(lens, device=dev)  # place of each sequence's last token
    total = 0
    for s in range(steps):
        live = torch.tensor([(s + b) % (N + 1) for b in range(B)], device=dev)
        drafts = torch.randint(0, V, (B, N), generator=g, device=dev)
        for i in range(s % N):  # some that are kept: what the model says itself
            drafts[:, i] = (step(last, drafts, live)[:, i] @ w["head"]).float().argmax(-1)
        x = step(last, drafts, live)
        logits = x @ w["head"]
        for b in range(B):
            tokens[b, last[b] + 1:last[b] + 1 + N] = drafts[b]
        want, cu = _whole(w, tokens, (last + live + 1).tolist(), dev)
        for b in range(B):
            n = int(live[b]) + 1
            near(x[b, :n], want[cu[b + 1] - n:cu[b + 1]])
        r = mk.verify_drafts(logits, drafts, torch.rand(B, N + 1, generator=g, device=dev), draft_lens=live, temperature=0.0)
        best = logits.float().argmax(-1)
        i = torch.arange(N, device=dev)
        kept = ((drafts == best[:, :N]) & (i < live[:, None])).long().cumprod(-1).sum(-1)
        assert torch.equal(r.accepted.long(), kept)
        assert torch.equal(r.tokens[row, kept], best[row, kept])
        total += int(kept.sum())
        # the kept drafts and the model's own token become the sequence
        for b in range(B):
            n = int(kept[b]) + 1
            tokens[b, last[b] + 1:last[b] + 1 + n] = r.tokens[b, :n]
        last = last + kept + 1
    assert total > steps  # drafts were kept, and others turned away
    score = mk.token_logprobs(logits[:, 0], best[:, 0])
    assert bool((score.logp > -20).all())


def _held(x, fmt):
    """fp64 rows as a cache of this format holds them."""
    x = x.double()
    if fmt == "bf16":
        return x.float().bfloat16().double()
    if fmt == "e4m3":
        top = x.float().abs().amax(-1, keepdim=True)
        s = torch.where(top > 0, top / torch.full_like(top, 448.0), torch.ones_like(top))
        return (x.float() / s).to(torch.float8_e4m3fn).double() * s.double()
    y = x.unflatten(-1, (-1, 32))
    power = torch.frexp(y.abs().amax(-1, keepdim=True))[1] - 3
    z = torch.ldexp(y, -power)
    step = torch.where(z.abs() < 2, 0.5, torch.where(z.abs() < 4, 1.0, 2.0)).double()
    return torch.ldexp(((z / step).round() * step).clamp(-6, 6), power).flatten(-2)


def _turned64(x, pos, freq):
    angle = (pos.double()[:, None, None].cpu() * freq.double().cpu())
    a, b = x.double().cpu().chunk(2, -1)
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1).to(x.device)


def _attended(q, k, v, seen):
    """fp64 attention of rows q (n, H, hd) over keys (m, Hkv, hd) where seen (n, m), and
    what bounds a kernel's error: the weights and the result are rounded to bf16 once
    each, at most 2^-8; exponents and fp32 sums add less than 2^-10."""
    G = q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(G, 1) for x in (k, v))
    s = (q.double()[:, None] * k).sum(-1).permute(2, 0, 1) * HD ** -0.5
    p = torch.softmax(s.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)  # (H, n, m)
    weigh = lambda y: torch.bmm(p, y.transpose(0, 1).contiguous()).transpose(0, 1)  # noqa: E731
    return weigh(v), weigh(v.abs()) * (2.0 ** -7 + 2.0 ** -10)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "e2m1"])
def test_speculative_steps_operator_by_operator(fmt, dev):
    """The loop above with each operator against fp64 on what it was given: the cache's
    rows are the keys turned to their own positions (those of the next position are far
    outside the bound), and each new token sees the tokens up to itself (one less, or
    one more, is outside the bound in every sequence that has one)."""
    from naylis_amd import mom_kernels as mk
    w = _weights(dev)
    g = torch.Generator(device=dev).manual_seed(2)
    prompts, steps = [37, 2, 130, 64], 4
    B, row = len(prompts), torch.arange(len(prompts), device=dev)
    width = -(-(max(prompts) + (steps + 1) * (N + 1)) // PAGE)
    tokens = torch.randint(0, V, (B, width * PAGE), generator=g, device=dev)
    table = torch.randperm(B * width + 1, generator=g, device=dev)[:B * width].view(B, width).int()
    caches = [mk.new_paged_cache(B * width + 1, HKV, PAGE, HD, dev, fp8=fmt == "e4m3", fp4=fmt == "e2m1") for _ in range(LAYERS)]

    def rows_of(c, rows, pos):
        at, off = table[rows.long(), pos.long() // PAGE].long(), pos.long() % PAGE
        return [x[at, :, off].double() for x in c.dequantize()]

    def appended(c, q, k, v, rows, pos):
        """Rotates and appends; tokens at position -1 are left out."""
        out = mk.paged_append_rope(c, q, k, v, w["freq"], table, pos, rows)
        far = lambda x, y: float((x - y).norm() / y.norm())  # noqa: E731
        assert far(out.double(), _turned64(q, pos, w["freq"])) < 2.0 ** -8
        live = pos >= 0
        got, at = rows_of(c, rows[live], pos[live]), pos[live]
        # (a value that fp32 puts on a border's other side is off by a step: a row in a
        # thousand, of whose norm that is an eighth at most)
        want = _held(_turned64(k[live], at, w["freq"]), fmt)
        assert far(got[0], want) < 2.0 ** -7 and far(got[1], _held(v[live], fmt)) < 2.0 ** -7
        assert far(_held(_turned64(k[live], at + 1, w["freq"]), fmt), want) > 2.0 ** -3
        return out

    def check(got, q, k, v, seen):
        want, bound = _attended(q, k, v, seen)
        assert bool(((got.double() - want).abs() <= bound + 1e-30).all())
        for off in (-1, 1):
            other = torch.zeros_like(seen)
            if off < 0:
                other[:, :-1] = seen[:, 1:]  # the token itself unseen
            else:
                other[:, 0], other[:, 1:] = True, seen[:, :-1]  # the next one too
            if bool((other != seen).any()):
                assert bool(((_attended(q, k, v, other)[0] - want).abs() > 2 * bound).any())

    lens = [n - 1 for n in prompts]
    cu, rows, pos = _places(lens, dev)
    x = w["embed"][tokens[rows.long(), pos.long()]]
    for c, lw in zip(caches, w["layers"]):
        def attend(q, k, v):
            q = appended(c, q, k, v, rows, pos)
            k, v = mk.paged_gather(c, table, cu, len(q))
            held = rows_of(c, rows, pos)
            assert torch.equal(k, held[0].float().bfloat16()) and torch.equal(v, held[1].float().bfloat16())
            out = mk.packed_attention(q, k, v, cu)
            for b in range(B):
                a, e = int(cu[b]), int(cu[b + 1])
                check(out[a:e], q[a:e], k[a:e], v[a:e], torch.ones(e - a, e - a, dtype=torch.bool, device=dev).tril())
            return out
        x = _layer(x, lw, attend)

    last = torch.tensor(lens, device=dev)
    for s in range(steps):
        live = torch.tensor([(s + b) % (N + 1) for b in range(B)], device=dev)
        drafts = torch.randint(0, V, (B, N), generator=g, device=dev)
        at = last[:, None] + torch.arange(N + 1, device=dev)
        at = torch.where(at <= (last + live)[:, None], at, -1).flatten().int()
        x = w["embed"][torch.cat([tokens[row, last][:, None], drafts], 1).flatten()]
        for c, lw in zip(caches, w["layers"]):
            def attend(q, k, v):
                q = appended(c, q, k, v, row.repeat_interleave(N + 1).int(), at).view(B, N + 1, H, HD)
                out = mk.paged_attention(q, c, table, last + live + 1, q_lens=live + 1)
                for b in range(B):
                    m, n = int(last[b] + live[b]) + 1, int(live[b]) + 1
                    i = torch.arange(m, device=dev)
                    k, v = rows_of(c, torch.full_like(i, b), i)
                    check(out[b, :n], q[b, :n], k, v, i <= i[m - n:, None])
                    assert not bool(out[b, n:].any())
                return out
            x = _layer(x, lw, attend)
        last = last + live + 1  # (all kept)
        tokens[row[:, None], last[:, None] - live[:, None] + torch.arange(N, device=dev)] = drafts


def test_speculative_operators_under_trace(dev):
    """Traced verifications run again on new inputs; the rotated append, whose results
    are also what it writes, refuses to be traced."""
    from naylis_amd import mom_kernels as mk
    g = torch.Generator(device=dev).manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    drafts = torch.randint(0, 50, (3, 2), generator=g, device=dev)
    lens, temps = torch.tensor([2, 1, 0], dtype=torch.int32, device=dev), torch.tensor([1.0, 0.0, 0.7], device=dev)
    for vocab in (50, 40000):  # one launch; more, with a workspace
        inputs = lambda: (rand(3, 3, vocab), torch.rand(3, 3, generator=g, device=dev), torch.softmax(rand(3, 2, vocab), -1))  # noqa: B023,E731
        for call in (lambda x, u, q: tuple(mk.verify_drafts(x, drafts, u, draft_probs=q, draft_lens=lens, temperature=temps)),
                     lambda x, u, q: tuple(mk.verify_drafts(x, drafts, u, temperature=0.5))):
            traced = torch.jit.trace(call, inputs(), check_trace=False)
            for _ in range(4):
                x = inputs()
                assert all(torch.equal(a, b) for a, b in zip(traced(*x), call(*x)))
    cache = mk.new_paged_cache(4, 2, 16, 64, dev, fp4=True)
    table, at = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2), torch.tensor([3, 4], dtype=torch.int32, device=dev)
    k = rand(2, 2, 64).bfloat16()
    with pytest.raises(RuntimeError, match="in place"):
        torch.jit.trace(lambda k: mk.paged_append_rope(cache, k, k, k, torch.ones(32, device=dev), table, at), (k,))

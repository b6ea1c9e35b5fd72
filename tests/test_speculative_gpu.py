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

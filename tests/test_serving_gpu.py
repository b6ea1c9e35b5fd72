"""The serving operators together, as a program uses them: a packed prompt pass
whose keys and values go into a paged cache, steps of one token over it, and
scores of the answers; and a policy update through packed attention and token
log probabilities."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, HKV, HD, V, LAYERS = 256, 4, 2, 64, 1000, 2


def _weights(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: (torch.randn(*s, generator=g, device=dev) * s[0] ** -0.5).bfloat16()  # noqa: E731
    return dict(embed=(torch.randn(V, D, generator=g, device=dev)).bfloat16(),
                layers=[dict(q=r(D, H * HD), k=r(D, HKV * HD), v=r(D, HKV * HD), o=r(H * HD, D)) for _ in range(LAYERS)],
                head=r(D, V))


def _layer(x, w, attend):
    h = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5)
    h = h.bfloat16()
    q, k, v = ((h @ w[n]).view(len(x), -1, HD) for n in "qkv")
    return x + attend(q, k, v).reshape(len(x), -1) @ w["o"]


def test_prompt_then_steps_match_the_whole(dev):
    """Hidden states of prompts of different lengths and of eight steps after
    them, each against the packed pass over the whole sequences so far."""
    from naylis_amd import mom_kernels as mk
    w = _weights(dev)
    g = torch.Generator(device=dev).manual_seed(1)
    prompts, steps, page = [37, 1, 130, 64], 8, 16
    B = len(prompts)
    tokens = torch.randint(0, V, (B, max(prompts) + steps), generator=g, device=dev)
    width = -(-tokens.shape[1] // page)
    table = torch.randperm(B * width + 1, generator=g, device=dev)[:B * width].view(B, width).int()

    def packed(lens, caches=None):
        """Rows of all sequences; with caches, their keys and values are appended."""
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
        rows = torch.repeat_interleave(torch.arange(B), torch.tensor(lens)).to(dev, torch.int32)
        pos = torch.cat([torch.arange(n) for n in lens]).to(dev, torch.int32)
        x = w["embed"][tokens[rows.long(), pos.long()]]
        for i, lw in enumerate(w["layers"]):
            def attend(q, k, v):
                if caches:
                    mk.paged_append(caches[i], k, v, table, pos, rows)
                return mk.packed_attention(q, k, v, cu)
            x = _layer(x, lw, attend)
        return x, [c - 1 for c in cu.tolist()[1:]]

    for fp8 in (False, True):
        caches = [mk.new_paged_cache(B * width + 1, HKV, page, HD, dev, fp8=fp8) for _ in range(LAYERS)]
        packed(prompts, caches)
        lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
        for step in range(steps):
            x = w["embed"][tokens[torch.arange(B, device=dev), lens.long()]]
            for i, lw in enumerate(w["layers"]):
                def attend(q, k, v):
                    mk.paged_append(caches[i], k, v, table, lens)
                    return mk.paged_attention(q, caches[i], table, lens + 1)
                x = _layer(x, lw, attend)
            lens = lens + 1
            whole, last = packed([n + step + 1 for n in prompts])
            want = whole[last].float()
            # each attention is within 2^-7 of itself on either side, each bf16
            # projection and sum a rounding more, over two layers; e4m3 rows are off
            # by at most 2^-4 of themselves, keys and values alike
            far = float((x.float() - want).norm() / want.norm())
            assert far < (2.0 ** -2 if fp8 else 2.0 ** -5), (fp8, step, far)
            if not fp8:
                a, b = (mk.token_logprobs(y.bfloat16() @ w["head"], tokens[:, 0], top=3) for y in (x, want))
                assert float((a.logp - b.logp).abs().max()) < 0.25 and a.top_ids.shape == (B, 3)


def test_policy_gradient_matches_fp64(dev):
    """Gradients of a packed layer's weights for logp and entropy of the tokens,
    against the same in fp64 autograd."""
    from naylis_amd import mom_kernels as mk
    w = _weights(dev)
    g = torch.Generator(device=dev).manual_seed(2)
    lens = [70, 5, 33]
    T = sum(lens)
    cu = torch.tensor([0, 70, 75, 108], dtype=torch.int32, device=dev)
    x = torch.randn(T, D, generator=g, device=dev).bfloat16()
    tok = torch.randint(0, V, (T,), generator=g, device=dev)
    adv = torch.randn(T, generator=g, device=dev)
    names = ("q", "k", "v", "o")
    params = [w["layers"][0][n].clone().requires_grad_() for n in names]

    def loss(ws, attend, logprobs):
        h = x.to(ws[0].dtype)
        q, k, v = ((h @ p).view(T, -1, HD) for p in ws[:3])
        y = h + attend(q, k, v).reshape(T, -1) @ ws[3]
        logp, entropy = logprobs(y @ w["head"].to(y.dtype))
        return (adv.to(logp.dtype) * logp).sum() + 0.1 * entropy.sum()

    def scored(z):
        r = mk.token_logprobs(z, tok)
        return r.logp, r.entropy

    def attend64(q, k, v):
        out = []
        for a, b in zip(cu.tolist(), cu.tolist()[1:]):
            s = q[a:b].transpose(0, 1) @ k[a:b].repeat_interleave(H // HKV, 1).permute(1, 2, 0).contiguous() * HD ** -0.5
            s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device=dev).triu(1), -math.inf)
            out.append((torch.softmax(s, -1) @ v[a:b].repeat_interleave(H // HKV, 1).transpose(0, 1).contiguous()).transpose(0, 1))
        return torch.cat(out)

    def scored64(z):
        lp = torch.log_softmax(z, -1)
        return lp.gather(1, tok[:, None])[:, 0], -(lp.exp() * lp).sum(-1)

    got = torch.autograd.grad(loss(params, lambda q, k, v: mk.packed_attention(q, k, v, cu), scored), params)
    exact = [p.detach().double().requires_grad_() for p in params]
    want = torch.autograd.grad(loss(exact, attend64, scored64), exact)
    for n, a, b in zip(names, got, want):
        # about eight bf16 roundings (2^-8 each) lie between the loss and a weight
        assert float((a.double() - b).norm() / b.norm()) < 8 * 2.0 ** -8, n


def test_operators_under_trace(dev):
    """Traced calls run again on new inputs; the append, whose result is what it
    writes, refuses to be traced."""
    from naylis_amd import mom_kernels as mk
    g = torch.Generator(device=dev).manual_seed(6)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()  # noqa: E731
    cu, tok = torch.tensor([0, 5, 20], dtype=torch.int32, device=dev), torch.arange(4, device=dev)
    cache = mk.new_paged_cache(4, 2, 16, 64, dev, fp8=True)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    lens = torch.tensor([20, 3], dtype=torch.int32, device=dev)
    for row in range(2):
        mk.paged_append(cache, rand(32, 2, 64), rand(32, 2, 64), table, torch.arange(32, device=dev),
                        torch.full((32,), row, device=dev))
    calls = [(lambda q, k, v: mk.packed_attention(q, k, v, cu), lambda: (rand(20, 4, 64), rand(20, 2, 64), rand(20, 2, 64))),
             (lambda x: tuple(mk.token_logprobs(x, tok, top=3)), lambda: (rand(4, 100),)),
             (lambda q: mk.paged_attention(q, cache, table, lens), lambda: (rand(2, 4, 64),))]
    for call, inputs in calls:
        traced, x = torch.jit.trace(call, inputs(), check_trace=False), inputs()
        got, want = traced(*x), call(*x)
        pairs = zip(got, want) if isinstance(want, tuple) else [(got, want)]
        assert all(torch.equal(a, b) for a, b in pairs)
    with pytest.raises(RuntimeError, match="in place"):
        torch.jit.trace(lambda k: mk.paged_append(cache, k, k, table, lens), (rand(2, 2, 64),))


def test_forward_mode_is_refused(dev):
    """A dual tensor (which needs no requires_grad), with and without reverse mode,
    raises in every operator that it reaches: no result without its tangent."""
    from torch.autograd import forward_ad

    from naylis_amd import mom_kernels as mk
    g = torch.Generator(device=dev).manual_seed(7)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()  # noqa: E731
    cu, tok = torch.tensor([0, 5, 20], dtype=torch.int32, device=dev), torch.arange(4, device=dev)
    bf, e4 = (mk.new_paged_cache(4, 2, 16, 64, dev, fp8=fp8) for fp8 in (False, True))
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    lens = torch.tensor([1, 2], dtype=torch.int32, device=dev)
    kv = lambda: (rand(2, 2, 64), rand(2, 2, 64))  # noqa: E731
    calls = [(lambda q, k, v: mk.packed_attention(q, k, v, cu), (rand(20, 4, 64), rand(20, 2, 64), rand(20, 2, 64))),
             (lambda x: mk.token_logprobs(x, tok), (rand(4, 100),)),
             (lambda x: mk.token_logprobs(x, tok, top=3), (rand(4, 100).float(),)),
             (lambda k, v: mk.paged_append(bf, k, v, table, lens), kv()),
             (lambda q, k, v: mk.paged_attention(q, mk.PagedCache(k, v), table, lens), (rand(2, 4, 64), bf.k, bf.v)),
             (lambda s, t: mk.paged_attention(rand(2, 4, 64), mk.PagedCache(e4.k, e4.v, s, t), table, lens),
              (e4.k_scale, e4.v_scale)),
             (lambda s, t: mk.paged_append(mk.PagedCache(e4.k, e4.v, s, t), *kv(), table, lens), (e4.k_scale, e4.v_scale))]
    for call, args in calls:
        call(*args)
        for i, a in enumerate(args):
            for grads in (False, True):
                with torch.set_grad_enabled(grads), forward_ad.dual_level():
                    dual = forward_ad.make_dual(a, torch.ones_like(a))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(*args[:i], dual, *args[i + 1:])
            with pytest.raises(RuntimeError):
                torch.func.jvp(lambda t: call(*args[:i], t, *args[i + 1:]), (a,), (torch.ones_like(a),))
    for i in range(2):  # nor a cache's scales that want a gradient
        for call, args in calls[-2:]:
            with pytest.raises(RuntimeError, match="no backward"):
                call(*(a.clone().requires_grad_(j == i) for j, a in enumerate(args)))

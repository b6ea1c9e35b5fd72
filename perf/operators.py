"""The serving and scoring operators of the package, as measurable cases.

A decoder's prompts run through ``packed_attention`` (sequences of different
lengths in one packed batch, grouped heads, forward and backward), their keys
and values go into a paged cache (``paged_append``), each new token attends to
that cache (``paged_attention``), and the answers are scored
(``token_logprobs``).  ``run`` is one pass through one of them: with ``own``
false in elementary fp32 torch operations, with it true through the package's
public entry points.  ``exact`` restates each in fp64, one sequence at a time.

Kinds, and the ranges they stand for:

  prompt   packed causal attention, forward: 1..24 sequences of 1..16384
           tokens, heads of 64 or 128, 1..8 query heads for a key head, with
           or without keys of earlier tokens before the prompt
  train    the same forward and backward, sequences up to 4096 tokens
  decode   one new token for each of 1..128 sequences over a cache of 1..131072
           tokens each, bf16 or e4m3, pages of 16..128 tokens
  append   keys and values of 1..16384 tokens into the cache, bf16 or e4m3
  score    log probabilities, entropies and top alternatives of 1..4096 rows
           of 1000..152000 logits, forward or forward and backward

Lengths of packed sequences are a text of comma-separated numbers.
"""
import math

import torch

own = False

DEV = "cuda"
KINDS = ("prompt", "train", "decode", "append", "score")


def listed():
    return [
        # a handful of short prompts, from one token up: launch latency
        dict(name="prompt_short", kind="prompt", lq="1,2,7,12,19,25,33,48,64,101", lk="", H=16, Hkv=16, hd=64),
        # chunks of prompts whose earlier tokens are in the cache already, one of a single token
        dict(name="prompt_continued", kind="prompt", lq="512,512,300,1,257,1024", lk="4096,700,300,2049,1281,3501",
             H=32, Hkv=8, hd=128),
        # one long document
        dict(name="prompt_long", kind="prompt", lq="16381", lk="", H=16, Hkv=4, hd=128),
        # a packed training batch of the 300M-class decoder's heads (16376 tokens)
        dict(name="train_packed", kind="train", lq="2048,2047,1021,3885,777,2048,1533,2969,48", lk="", H=16, Hkv=16,
             hd=64),
        # a packed training batch with grouped heads of 128
        dict(name="train_grouped", kind="train", lq="4093,2500,1100,499", lk="", H=32, Hkv=8, hd=128),
        # one user's next token after a short prompt
        dict(name="decode_one", kind="decode", B=1, longest=500, H=16, Hkv=16, hd=64, page=16, fp8=False),
        # a serving batch at ragged lengths
        dict(name="decode_batch", kind="decode", B=64, longest=4096, H=32, Hkv=8, hd=128, page=32, fp8=False),
        # a few very long contexts over an e4m3 cache
        dict(name="decode_long_fp8", kind="decode", B=3, longest=131072, H=32, Hkv=8, hd=128, page=64, fp8=True),
        # a serving batch's new keys and values into an e4m3 cache
        dict(name="append_step", kind="append", T=64, seqs=64, longest=1024, Hkv=8, hd=128, page=16, fp8=True),
        # a packed prompt's keys and values into a bf16 cache
        dict(name="append_prompt", kind="append", T=8191, seqs=5, longest=2048, Hkv=8, hd=128, page=16, fp8=False),
        # a serving batch's answers with their twenty likeliest alternatives
        dict(name="score_step", kind="score", N=64, V=32768, top=20, dtype="bf16", train=False),
        # log probabilities and entropies of a policy update, with their gradient, at an odd vocabulary
        dict(name="score_train", kind="score", N=4096, V=50001, top=0, dtype="bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(lens):
    return ",".join(str(n) for n in lens)


def _heads(rng):
    H = rng.choice([4, 8, 16, 32])
    return dict(H=H, Hkv=max(1, H // rng.choice([1, 2, 4, 8])), hd=rng.choice([64, 128]))


def _drawn(rng, kind):
    if kind in ("prompt", "train"):
        n, longest = _log_int(rng, 1, 24), _log_int(rng, 16, 4096 if kind == "train" else 16384)
        lq = [longest] + [_log_int(rng, 1, longest) for _ in range(n - 1)]
        rng.shuffle(lq)
        lk = [a + rng.choice([0, _log_int(rng, 1, longest)]) for a in lq] if kind == "prompt" and rng.random() < 0.4 else []
        return dict(kind=kind, lq=_text(lq), lk=_text(lk), **_heads(rng))
    if kind == "decode":
        return dict(kind=kind, B=_log_int(rng, 1, 128), longest=_log_int(rng, 1, 131072), page=rng.choice([16, 32, 64, 128]),
                    fp8=rng.random() < 0.5, **_heads(rng))
    if kind == "append":
        seqs, h = _log_int(rng, 1, 64), _heads(rng)
        longest = _log_int(rng, 16, 4096)
        return dict(kind=kind, T=min(seqs * longest, _log_int(rng, 1, 16384)), seqs=seqs, longest=longest, Hkv=h["Hkv"],
                    hd=h["hd"], page=rng.choice([16, 32, 64, 128]), fp8=rng.random() < 0.5)
    return dict(kind=kind, N=_log_int(rng, 1, 4096), V=_log_int(rng, 1000, 152000), top=rng.choice([0, 1, 5, 20]),
                dtype=rng.choice(["bf16", "bf16", "f32"]), train=rng.random() < 0.5)


def _small_enough(case):
    """No more work than the listed cases, and plain forms that fit the card three times over."""
    w = work(case)
    if case["kind"] in ("prompt", "train"):
        lq, lk = _lens(case)
        padded = len(lq) * max(lq) * max(lk) * case["H"]
        return w["flops"] <= 1.05e12 and padded <= (2.3e9 if case["kind"] == "train" else 4.4e9)
    if case["kind"] == "score":
        return case["N"] * case["V"] <= (4096 * 50001 if case["top"] == 0 else 1e8)
    tokens = case["longest"] * case.get("B", case.get("seqs"))
    return tokens * case["Hkv"] * case["hd"] <= 4.1e8


def draw(rng):
    kind = rng.choice(KINDS)
    while True:
        case = _drawn(rng, kind)
        if _small_enough(case):
            return case


def _lens(case):
    lq = [int(x) for x in case["lq"].split(",")]
    return lq, [int(x) for x in case["lk"].split(",")] if case["lk"] else lq


def _decode_lens(case):
    """Cache lengths from the longest down to an eighth of it, unevenly."""
    return [max(1, case["longest"] - (i * i * 7919) % max(1, case["longest"] * 7 // 8)) for i in range(case["B"])]


def _append_lens(case):
    """How many of the T tokens each sequence gets."""
    T, n = case["T"], case["seqs"]
    return [T // n + (1 if i < T % n else 0) for i in range(n)]


# ---- inputs ------------------------------------------------------------------


def _offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).to(DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _quantize(x):
    """Rows as e4m3 codes with one fp32 scale: max|row| / 448, 1 for a row of zeros."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    return (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _cache(g, pages, case):
    """Key and value pages (pages, Hkv, page, hd) as earlier steps left them, and their scales (None for bf16)."""
    shape = (pages, case["Hkv"], case["page"], case["hd"])
    k, v = _randn(g, *shape), _randn(g, *shape)
    if not case["fp8"]:
        return k, v, None, None
    (k, ks), (v, vs) = _quantize(k), _quantize(v)
    return k, v, ks, vs


def _table(g, lens, page):
    """Each sequence's pages, in no order, -1 behind its last."""
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(need) + 3, generator=g, device=DEV).to(torch.int32)
    width = max(need)
    at = torch.arange(width, device=DEV)[None] + (torch.tensor(need).cumsum(0) - torch.tensor(need)).to(DEV)[:, None]
    live = torch.arange(width, device=DEV)[None] < torch.tensor(need).to(DEV)[:, None]
    return torch.where(live, ids[at.clamp(max=ids.numel() - 1)], -1).contiguous(), sum(need) + 3


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = dict(case=dict(case))
    if kind in ("prompt", "train"):
        lq, lk = _lens(case)
        T, Tk, H, Hkv, hd = sum(lq), sum(lk), case["H"], case["Hkv"], case["hd"]
        s.update(q=_randn(g, T, H, hd, std=1.5), k=_randn(g, Tk, Hkv, hd), v=_randn(g, Tk, Hkv, hd), mq=max(lq),
                 mk=max(lk), cu_q=_offsets(lq), scale=hd ** -0.5)
        s["cu_k"] = _offsets(lk) if case["lk"] else s["cu_q"]
        if kind == "train":
            for n in "qkv":
                s[n].requires_grad_()
            s["dout"] = _randn(g, T, H, hd)
    elif kind == "decode":
        lens = _decode_lens(case)
        table, pages = _table(g, lens, case["page"])
        s.update(q=_randn(g, case["B"], case["H"], case["hd"], std=1.5), cache=_cache(g, pages, case), table=table,
                 lens=torch.tensor(lens, dtype=torch.int32).to(DEV), scale=case["hd"] ** -0.5)
    elif kind == "append":
        table, pages = _table(g, [case["longest"]] * case["seqs"], case["page"])
        add = _append_lens(case)
        start = torch.rand(case["seqs"], generator=g, device=DEV)
        room = torch.tensor([case["longest"] - a for a in add]).to(DEV)
        first = (start * (room + 1)).long().clamp(max=room)
        rows = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(add)).to(DEV)
        within = torch.arange(case["T"], device=DEV) - _offsets(add).long()[rows]
        s.update(cache=_cache(g, pages, case), table=table, rows=rows.to(torch.int32),
                 positions=(first[rows] + within).to(torch.int32), k=_randn(g, case["T"], case["Hkv"], case["hd"]),
                 v=_randn(g, case["T"], case["Hkv"], case["hd"]))
    else:
        N, V = case["N"], case["V"]
        x = _randn(g, N, V, std=2.0, dtype=torch.float32)
        hot = torch.randint(0, V, (N, 8), generator=g, device=DEV)  # a few likely tokens in each row
        x.scatter_add_(1, hot, torch.rand(N, 8, generator=g, device=DEV) * 12)
        x[:, V - V // 500:] = -math.inf  # columns that pad the vocabulary
        tokens = torch.where(torch.rand(N, generator=g, device=DEV) < 0.7, hot[:, 0], hot[:, 1]).clamp(max=V - V // 500 - 1)
        s.update(logits=x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32), tokens=tokens)
        if case["train"]:
            s["logits"].requires_grad_()
            s["g_logp"] = torch.randn(N, generator=g, device=DEV) / N
            s["g_entropy"] = torch.full((N,), -0.01 / N, device=DEV)
    return s


# ---- plain forms -------------------------------------------------------------


def _pad(x, cu, longest):
    """Packed rows (T, H, hd) as (n, H, longest, hd) fp32, and each sequence's length."""
    start, end = cu[:-1].long(), cu[1:].long()
    at = (start[:, None] + torch.arange(longest, device=x.device)).clamp(max=x.shape[0] - 1)
    return x[at].float().transpose(1, 2), end - start


def _unpad(x, cu, rows, dtype):
    """(n, H, longest, hd) back to packed rows."""
    t = torch.arange(rows, device=x.device)
    seq = torch.searchsorted(cu[1:].long().contiguous(), t, right=True)
    return x[seq, :, t - cu.long()[seq]].to(dtype)


def _plain_weights(qf, kf, lq, lk, scale):
    """softmax over the keys that each query may see; qf (n, Hkv, G, mq, hd), kf (n, Hkv, mk, hd)."""
    n, Hkv, G, mq, hd = qf.shape
    mk = kf.shape[2]
    s = (qf.reshape(n, Hkv, G * mq, hd) @ kf.transpose(-1, -2).contiguous()).mul_(scale).view(n, Hkv, G, mq, mk)
    i, j = torch.arange(mq, device=qf.device)[None, :, None], torch.arange(mk, device=qf.device)[None, None]
    lq, lk = lq[:, None, None], lk[:, None, None]
    hidden = ((j > i + lk - lq) | (j >= lk) | (i >= lq))[:, None, None]
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    return s.div_(s.sum(-1, keepdim=True).clamp(min=1e-38))


def _plain_attention(s):
    q, k, v = (s[n].detach() for n in "qkv")
    (T, H, hd), Hkv = q.shape, k.shape[1]
    qf, lq = _pad(q, s["cu_q"], s["mq"])
    (kf, lk), (vf, _) = _pad(k, s["cu_k"], s["mk"]), _pad(v, s["cu_k"], s["mk"])
    n, G, mq, mk = qf.shape[0], H // Hkv, s["mq"], s["mk"]
    qf = qf.reshape(n, Hkv, G, mq, hd)
    p = _plain_weights(qf, kf, lq, lk, s["scale"])
    o = p.view(n, Hkv, G * mq, mk) @ vf.contiguous()
    out = _unpad(o.view(n, H, mq, hd), s["cu_q"], T, q.dtype)
    if "dout" not in s:
        return out
    # rows past a sequence's end have no weights, so whatever stands there adds nothing
    df = _pad(s["dout"], s["cu_q"], mq)[0].reshape(n, Hkv, G * mq, hd)
    pt = p.view(n, Hkv, G * mq, mk)
    dv = pt.transpose(-1, -2).contiguous() @ df
    ds = df @ vf.transpose(-1, -2).contiguous()
    ds.sub_((df * o).sum(-1, keepdim=True)).mul_(pt).mul_(s["scale"])
    dq = (ds @ kf.contiguous()).view(n, H, mq, hd)
    dk = ds.transpose(-1, -2).contiguous() @ qf.reshape(n, Hkv, G * mq, hd)
    return (out, _unpad(dq, s["cu_q"], T, q.dtype), _unpad(dk, s["cu_k"], k.shape[0], k.dtype),
            _unpad(dv, s["cu_k"], v.shape[0], v.dtype))


def _plain_pages(pages, scale, table):
    """The table's pages as (B, Hkv, tokens, hd) fp32."""
    x = pages[table.long().clamp(min=0)]
    x = x.float() if scale is None else x.view(torch.float8_e4m3fn).float() * scale[table.long().clamp(min=0)][..., None]
    B, P, Hkv, page, hd = x.shape
    return x.transpose(1, 2).reshape(B, Hkv, P * page, hd)


def _plain_decode(s):
    q, (kp, vp, ks, vs) = s["q"], s["cache"]
    B, H, hd = q.shape
    k = _plain_pages(kp, ks, s["table"])
    Hkv = k.shape[1]
    w = (q.float().view(B, Hkv, H // Hkv, hd) @ k.transpose(-1, -2).contiguous()).mul_(s["scale"])
    del k
    w.masked_fill_((torch.arange(w.shape[-1], device=q.device)[None] >= s["lens"][:, None])[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    w.div_(w.sum(-1, keepdim=True).clamp(min=1e-38))
    return (w @ _plain_pages(vp, vs, s["table"])).view(B, H, hd).to(q.dtype)


def _plain_append(s):
    kp, vp, ks, vs = s["cache"]
    page = kp.shape[2]
    at, off = s["table"][s["rows"].long(), s["positions"].long() // page].long(), s["positions"].long() % page
    if ks is None:
        kp[at, :, off], vp[at, :, off] = s["k"], s["v"]
    else:
        (kp[at, :, off], ks[at, :, off]), (vp[at, :, off], vs[at, :, off]) = _quantize(s["k"]), _quantize(s["v"])
    return _cache_values(s["cache"])


def _cache_values(cache):
    """The cache itself; e4m3 codes as the numbers they stand for."""
    k, v, ks, vs = cache
    return (k, v) if ks is None else (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs)


def _plain_score(s):
    x, tok = s["logits"].detach().float(), s["tokens"]
    lp = x - x.amax(-1, keepdim=True)
    lp = lp - lp.exp().sum(-1, keepdim=True).log()
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    out = [lp.gather(1, tok[:, None])[:, 0], entropy]
    if s["case"]["top"]:
        best = torch.sort(s["logits"].detach(), dim=-1, descending=True, stable=True)[1][:, :s["case"]["top"]]
        out += [best, lp.gather(1, best)]
    if s["case"]["train"]:
        gl, ge = s["g_logp"][:, None], s["g_entropy"][:, None]
        d = torch.where(p > 0, p * (lp + entropy[:, None]), 0.0).mul_(-ge).sub_(p.mul_(gl))
        d.scatter_add_(1, tok[:, None], gl)
        out.append(d.to(s["logits"].dtype))
    return out


def _plain(s):
    kind = s["case"]["kind"]
    if kind in ("prompt", "train"):
        return _plain_attention(s)
    return {"decode": _plain_decode, "append": _plain_append, "score": _plain_score}[kind](s)


# ---- the package's entry points ------------------------------------------------


def _own(s):
    from naylis_amd import mom_kernels as mk
    kind = s["case"]["kind"]
    if kind in ("prompt", "train"):
        out = mk.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], scale=s["scale"])
        if kind == "prompt":
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    if kind == "decode":
        return mk.paged_attention(s["q"], mk.PagedCache(*s["cache"]), s["table"], s["lens"], scale=s["scale"])
    if kind == "append":
        mk.paged_append(mk.PagedCache(*s["cache"]), s["k"], s["v"], s["table"], s["positions"], s["rows"])
        return _cache_values(s["cache"])
    r = mk.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    out = [r.logp.detach(), r.entropy.detach()]
    if s["case"]["top"]:
        out += [r.top_ids, r.top_logp]
    if s["case"]["train"]:
        out += torch.autograd.grad((r.logp, r.entropy), s["logits"], (s["g_logp"], s["g_entropy"]))
    return out


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- work --------------------------------------------------------------------


def _pairs(lq, lk):
    """(query, key) pairs of the causal masks, the last query at the last key."""
    hidden = [min(a, max(0, a - b)) for a, b in zip(lq, lk)]  # queries before the first key
    return sum((a - h) * (b - a + h + 1 + b) // 2 for a, b, h in zip(lq, lk, hidden))


def work(case):
    kind = case["kind"]
    if kind in ("prompt", "train"):
        lq, lk = _lens(case)
        n = _pairs(lq, lk) * case["H"] * case["hd"]
        rows = sum(lq) * case["H"] * case["hd"] * 2, sum(lk) * case["Hkv"] * case["hd"] * 2
        if kind == "prompt":
            return {"bytes": 2 * rows[0] + 2 * rows[1], "flops": 4 * n}
        return {"bytes": 4 * rows[0] + 4 * rows[1], "flops": 14 * n}
    row = case.get("Hkv", 0) * (case.get("hd", 0) + 4 if case.get("fp8") else 2 * case.get("hd", 0))
    if kind == "decode":
        tokens, q = sum(_decode_lens(case)), case["B"] * case["H"] * case["hd"]
        return {"bytes": 2 * tokens * row + 4 * q, "flops": 4 * tokens * case["H"] * case["hd"]}
    if kind == "append":
        return {"bytes": 2 * case["T"] * (row + case["Hkv"] * case["hd"] * 2), "flops": 0}
    cells = case["N"] * case["V"]
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": cells * size * (2 if case["train"] else 1), "flops": cells * (8 if case["train"] else 4)}


# ---- fp64 statements -----------------------------------------------------------


def _exact_attention(s):
    lq, lk = _lens(s["case"])
    q, k, v = (s[n].detach() for n in "qkv")
    Hkv, G = k.shape[1], q.shape[1] // k.shape[1]
    res = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (q, q, k, v)]
    a = b = 0
    for nq, nk in zip(lq, lk):
        see = torch.ones(nq, nk, dtype=torch.bool, device=DEV).tril(nk - nq)
        for h in range(G * Hkv):
            c = h // G
            x, y, z = q[a:a + nq, h].double(), k[b:b + nk, c].double(), v[b:b + nk, c].double()
            w = torch.softmax((x @ y.T * s["scale"]).masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
            o = w @ z
            res[0][a:a + nq, h] = o
            if "dout" in s:
                d = s["dout"][a:a + nq, h].double()
                res[3][b:b + nk, c] += w.T @ d
                w = w * (d @ z.T - (d * o).sum(-1, keepdim=True)) * s["scale"]
                res[1][a:a + nq, h] = w @ y
                res[2][b:b + nk, c] += w.T @ x
        a, b = a + nq, b + nk
    return tuple(res) if "dout" in s else res[0]


def _exact_decode(s):
    q, (kp, vp, ks, vs) = s["q"].double(), s["cache"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    G, page = q.shape[1] // kp.shape[1], kp.shape[2]
    for b, n in enumerate(_decode_lens(s["case"])):
        ids = s["table"][b, :-(-n // page)].long()
        for c in range(kp.shape[1]):
            k, v = kp[ids, c], vp[ids, c]
            if ks is None:
                k, v = k.double(), v.double()
            else:
                k = k.view(torch.float8_e4m3fn).double() * ks[ids, c].double()[..., None]
                v = v.view(torch.float8_e4m3fn).double() * vs[ids, c].double()[..., None]
            k, v = k.reshape(-1, k.shape[-1])[:n], v.reshape(-1, v.shape[-1])[:n]
            out[b, c * G:(c + 1) * G] = torch.softmax(q[b, c * G:(c + 1) * G] @ k.T * s["scale"], -1) @ v
    return out


def _exact_append(s):
    kp, vp, ks, vs = s["cache"]
    page = kp.shape[2]
    pos = s["positions"].long()
    slot = s["table"][s["rows"].long(), pos // page].long() * page + pos % page
    res = []
    for pages, scale, new in ((kp, ks, s["k"].double()), (vp, vs, s["v"].double())):
        x = (pages if scale is None else pages.view(torch.float8_e4m3fn)).double().transpose(1, 2).contiguous()
        if scale is not None:
            top = new.abs().amax(-1)
            new_scale = torch.where(top > 0, top / 448, 1.0)
            new = new / new_scale[..., None]
            y = scale.double().transpose(1, 2).contiguous()
            y.view(-1, y.shape[-1])[slot] = new_scale
            res.append(y.transpose(1, 2))
        x.view(-1, *x.shape[2:])[slot] = new
        res.append(x.transpose(1, 2))
    return tuple(res) if ks is None else (res[1], res[3], res[0], res[2])


def _exact_score(s):
    x, tok, top = s["logits"].detach().double(), s["tokens"], s["case"]["top"]
    at = torch.arange(x.shape[0], device=DEV)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[:, None])
    entropy = lse - (p * x.clamp(min=-1e300)).sum(-1)
    out = [x[at, tok] - lse, entropy]
    if top:
        out += [None, torch.topk(x, top, -1)[0] - lse[:, None]]
    if s["case"]["train"]:
        d = -p * (s["g_logp"].double() + s["g_entropy"].double() * (entropy - lse))[:, None]
        d -= p * x.clamp(min=-1e300) * s["g_entropy"].double()[:, None]
        d[at, tok] += s["g_logp"].double()
        out.append(d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("prompt", "train"):
        return _exact_attention(s)
    return {"decode": _exact_decode, "append": _exact_append, "score": _exact_score}[kind](s)

"""The operators of speculative decoding over a small cache, as measurable cases.

A serving step with drafted tokens runs: the new tokens' queries and keys are
rotated to their positions and the keys and values go into a paged cache
(``paged_append_rope``), the queries of a sequence's few new tokens read that
cache (``paged_attention`` over several tokens, pages in 4 bits among them),
and the drafts are held against the logits that come of it
(``verify_drafts``).  A chunk of a prompt does the first step with many tokens
and takes the sequence's keys and values back dense (``paged_gather``), for
``packed_attention``.  ``run`` is one pass: with ``own`` false in elementary
torch operations, with it true through the package's public entry points.
``exact`` restates each in fp64.

Kinds, and the ranges they stand for:

  append   1..16384 tokens rotated and into the cache, at positions up to
           131071; pages of bf16 or e4m3, whole or half rotated heads
  extend   the same into sequences of 16..16384 tokens in all, pages of any of
           the three types, then those sequences' keys and values dense in bf16
  attend   1..8 new tokens of 1..128 sequences over a cache of 1..131072 tokens
           each: pages of 4 bits (e2m1, a power of two for 32 values), several
           tokens over bf16 and e4m3 pages too
  verify   0..8 drafts of 1..128 sequences against 1000..152000 logits, drawn
           from given probabilities or by a rule, some rows greedy
"""
import math

import torch

own = False

DEV = "cuda"
KINDS = ("append", "extend", "attend", "verify")
FORMATS = ("bf16", "e4m3", "e2m1")
FAR = 131072  # positions


def listed():
    return [
        # a serving batch's step with three drafts each, positions far apart, into an e4m3 cache
        dict(name="append_drafts", kind="append", T=256, seqs=64, H=32, Hkv=8, hd=128, rot=128, page=16, fmt="e4m3"),
        # a packed prompt's tokens at once into a bf16 cache
        dict(name="append_prompt", kind="append", T=8191, seqs=5, H=32, Hkv=8, hd=128, rot=128, page=16, fmt="bf16"),
        # chunks of prompts behind their earlier tokens, in 4 bits
        dict(name="extend_chunks", kind="extend", T=2048, seqs=4, longest=4093, H=32, Hkv=8, hd=128, rot=128, page=32,
             fmt="e2m1"),
        # the 300M-class decoder's heads, half of each rotated, one long document's last chunk
        dict(name="extend_document", kind="extend", T=1021, seqs=1, longest=16381, H=16, Hkv=16, hd=64, rot=32, page=64,
             fmt="e4m3"),
        # one user's next token after a short prompt
        dict(name="attend_one", kind="attend", B=1, N=1, longest=500, H=16, Hkv=16, hd=64, page=16, fmt="e2m1"),
        # a serving batch at ragged lengths, a token each
        dict(name="attend_batch", kind="attend", B=64, N=1, longest=4096, H=32, Hkv=8, hd=128, page=32, fmt="e2m1"),
        # a few very long contexts in 4 bits with three drafts each
        dict(name="attend_long_drafts", kind="attend", B=3, N=4, longest=131072, H=32, Hkv=8, hd=128, page=64, fmt="e2m1"),
        # a serving batch with up to four drafts each over a bf16 cache
        dict(name="attend_drafts", kind="attend", B=32, N=5, longest=8191, H=32, Hkv=8, hd=128, page=16, fmt="bf16"),
        # one user's three drafts found by a rule (no probabilities of theirs)
        dict(name="verify_one", kind="verify", B=1, N=3, V=32768, dtype="bf16", probs="none", greedy=False),
        # a serving batch's drafts of a small model, at an odd vocabulary
        dict(name="verify_batch", kind="verify", B=64, N=4, V=50001, dtype="bf16", probs="f32", greedy=False),
        # a long vocabulary, many drafts, every fourth sequence greedy
        dict(name="verify_wide", kind="verify", B=48, N=7, V=151999, dtype="bf16", probs="bf16", greedy=True),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    H = rng.choice([4, 8, 16, 32])
    return dict(H=H, Hkv=max(1, H // rng.choice([1, 2, 4, 8])), hd=rng.choice([64, 128]))


def _drawn(rng, kind):
    page = rng.choice([16, 32, 64, 128])
    if kind in ("append", "extend"):
        h, seqs = _heads(rng), _log_int(rng, 1, 64)
        h["rot"] = h["hd"] // rng.choice([1, 1, 2])
        if kind == "append":
            return dict(kind=kind, T=_log_int(rng, 1, 16384), seqs=seqs, page=page, fmt=rng.choice(FORMATS[:2]), **h)
        longest = _log_int(rng, 16, 16384)
        return dict(kind=kind, T=_log_int(rng, 1, seqs * longest), seqs=seqs, longest=longest, page=page,
                    fmt=rng.choice(FORMATS), **h)
    if kind == "attend":
        N = rng.choice([1, 1, 2, 3, 4, 5, 6, 8])
        return dict(kind=kind, B=_log_int(rng, 1, 128), N=N, longest=_log_int(rng, 1, 131072), page=page,
                    fmt="e2m1" if N == 1 else rng.choice(FORMATS), **_heads(rng))
    return dict(kind=kind, B=_log_int(rng, 1, 128), N=rng.choice([0, 1, 2, 3, 4, 5, 7, 8]), V=_log_int(rng, 1000, 152000),
                dtype=rng.choice(["bf16", "bf16", "f32"]), probs=rng.choice(["none", "f32", "bf16"]),
                greedy=rng.random() < 0.3)


def _small_enough(case):
    """No more work than the listed cases, and plain forms that fit the card three times over."""
    kind = case["kind"]
    if kind == "append":
        return case["T"] * (case["H"] + 2 * case["Hkv"]) * case["hd"] <= 8191 * 48 * 128
    if kind == "extend":
        return (case["T"] <= 16384 and case["seqs"] * case["longest"] <= 65536
                and work(case)["bytes"] <= 1.13e8)
    if kind == "attend":
        w = work(case)
        return (case["longest"] * case["B"] * case["Hkv"] * case["hd"] <= 4.1e8 and w["flops"] <= 2.3e10
                and w["bytes"] <= 5.5e8)
    return case["B"] * (case["N"] + 1) * case["V"] <= 48 * 8 * 151999 and work(case)["bytes"] <= 1.16e8


def draw(rng):
    kind = rng.choice(KINDS)
    while True:
        case = _drawn(rng, kind)
        if _small_enough(case):
            return case


def _cache_lens(case):
    """Cache lengths from the longest down to an eighth of it, unevenly."""
    return [max(1, case["longest"] - (i * i * 7919) % max(1, case["longest"] * 7 // 8)) for i in range(case["B"])]


def _shares(case):
    """How many of the T tokens each sequence gets."""
    T, n = case["T"], case["seqs"]
    return [T // n + (1 if i < T % n else 0) for i in range(n)]


def _ends(case):
    """Lengths of the sequences of a chunk with it, from the longest down to an eighth of it, unevenly."""
    return [max(a, case["longest"] - (i * i * 7919) % max(1, case["longest"] * 7 // 8)) for i, a in enumerate(_shares(case))]


def _live(case):
    """Live queries or drafts of each sequence: all of them for two in three, fewer for the others."""
    return [case["N"] - (i % 3 == 2) * (i % (case["N"] or 1)) for i in range(case["B"])]


# ---- inputs ------------------------------------------------------------------


def _offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).to(DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 29)


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _quantize(x, fmt):
    """Rows fp32 as codes and scales: e4m3 with max|row| / 448 in fp32 (1 for a row of zeros), or pairs of e2m1 in a
    byte with a power of two for 32 values (its exponent + 127 in a byte): that of the largest one over 4."""
    if fmt == "e4m3":
        top = x.abs().amax(-1)
        scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
        return (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale
    x = x.unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    byte = torch.where(top > 0, torch.frexp(top)[1] + 124, 1).clamp(min=1)  # frexp: top = m 2^e, m in [1/2, 1)
    y = torch.ldexp(x, (127 - byte)[..., None])
    a = y.abs()  # to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6, ties to the even code
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = (code | (torch.signbit(y).int() << 3)).flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] | (code[..., 1] << 4)).to(torch.uint8), byte.to(torch.uint8)


def _cache(g, pages, case):
    """Key and value pages (pages, Hkv, page, hd) as earlier steps left them, and their scales (None for bf16)."""
    shape = (pages, case["Hkv"], case["page"], case["hd"])
    if case["fmt"] == "e2m1":
        codes = [torch.randint(0, 256, shape[:3] + (shape[3] // 2,), generator=g, device=DEV, dtype=torch.uint8)
                 for _ in range(2)]
        scales = [torch.randint(124, 127, shape[:3] + (shape[3] // 32,), generator=g, device=DEV, dtype=torch.uint8)
                  for _ in range(2)]
        return (*codes, *scales)
    k, v = _randn(g, *shape), _randn(g, *shape)
    if case["fmt"] == "bf16":
        return k, v, None, None
    (k, ks), (v, vs) = _quantize(k.float(), "e4m3"), _quantize(v.float(), "e4m3")
    return k, v, ks, vs


def _table(g, first, end, page, tokens):
    """Pages of the tokens first[b] .. end[b] - 1 of each sequence, in no order, -1 elsewhere; how many there are (and
    some more) where none has over `tokens` tokens."""
    width = max(1, -(-tokens // page))
    at = torch.arange(width)[None]
    live = (at >= torch.tensor(first)[:, None] // page) & (at * page < torch.tensor(end)[:, None])
    pages = sum((e - f) // page + 2 for f, e in zip(first, end))
    ids = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    n, live = int(live.sum()), live.to(DEV)
    table = torch.full(live.shape, -1, dtype=torch.int32, device=DEV)
    table[live] = ids[:n]
    return table, pages


def _prepare_append(s, g, case):
    T, H, Hkv, hd = case["T"], case["H"], case["Hkv"], case["hd"]
    add = _shares(case)
    if case["kind"] == "append":  # anywhere; pages of earlier tokens do not matter
        start = torch.rand(case["seqs"], generator=g, device=DEV).cpu().tolist()
        first = held = [int(u * (FAR - a + 1)) for u, a in zip(start, add)]
        end = [f + a for f, a in zip(first, add)]
    else:
        end, held = _ends(case), [0] * len(add)
        first = [e - a for e, a in zip(end, add)]
    table, pages = _table(g, held, end, case["page"], case.get("longest", FAR))
    rows = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(add)).to(DEV)
    within = torch.arange(T, device=DEV) - _offsets(add).long()[rows]
    half = case["rot"] // 2
    s.update(cache=_cache(g, pages, case), table=table, rows=rows.to(torch.int32),
             positions=(torch.tensor(first).to(DEV)[rows] + within).to(torch.int32), q=_randn(g, T, H, hd, std=1.5),
             k=_randn(g, T, Hkv, hd), v=_randn(g, T, Hkv, hd),
             inv_freq=(500000.0 ** (-torch.arange(half, device=DEV).double() / half)).float())
    if case["kind"] == "extend":
        s.update(cu=_offsets(end), total=sum(end))


def _prepare_verify(s, g, case):
    B, N, V = case["B"], case["N"], case["V"]
    x = _randn(g, B, N + 1, V, std=2.0, dtype=torch.float32)
    hot = torch.randint(0, V - V // 500, (B, N + 1, 8), generator=g, device=DEV)  # a few likely tokens in each row
    x.scatter_add_(2, hot, 6 + torch.rand(B, N + 1, 8, generator=g, device=DEV) * 8)
    x[..., V - V // 500:] = -math.inf  # columns that pad the vocabulary
    if case["probs"] == "none":
        s["draft_probs"] = None
    else:  # another model's opinion of the same text
        y = x[:, :N] + _randn(g, B, N, V, std=0.7, dtype=torch.float32)
        s["draft_probs"] = torch.softmax(y, -1).to(torch.float32 if case["probs"] == "f32" else torch.bfloat16)
    best = x[:, :N].argmax(-1)
    likely = torch.rand(B, N, generator=g, device=DEV) < 0.7
    s.update(logits=x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32),
             drafts=torch.where(likely, best, hot[:, :N, 0]), uniforms=torch.rand(B, N + 1, generator=g, device=DEV),
             draft_lens=torch.tensor(_live(case), dtype=torch.int32).to(DEV),
             temperature=0.5 + torch.rand(B, generator=g, device=DEV))
    if case["greedy"]:
        s["temperature"][::4] = 0.0


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=dict(case))
    if case["kind"] in ("append", "extend"):
        _prepare_append(s, g, case)
    elif case["kind"] == "attend":
        lens, B, N = _cache_lens(case), case["B"], case["N"]
        table, pages = _table(g, [0] * B, lens, case["page"], max(lens))
        shape = (B, case["H"], case["hd"]) if N == 1 else (B, N, case["H"], case["hd"])
        s.update(q=_randn(g, *shape, std=1.5), cache=_cache(g, pages, case), table=table,
                 lens=torch.tensor(lens, dtype=torch.int32).to(DEV), scale=case["hd"] ** -0.5,
                 live=None if N == 1 else torch.tensor(_live(case), dtype=torch.int32).to(DEV))
    else:
        _prepare_verify(s, g, case)
    return s


# ---- plain forms -------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_PAIRS = [(s * a, t * b) for t in (1, -1) for b in _E2M1 for s in (1, -1) for a in _E2M1]  # low four bits first


def _values(codes, scale):
    """The numbers that cache rows stand for, fp32."""
    if scale is None:
        return codes.float()
    if scale.dtype == torch.float32:
        return codes.view(torch.float8_e4m3fn).float() * scale[..., None]
    x = torch.tensor(_PAIRS, device=codes.device)[codes.long()].flatten(-2)
    return torch.ldexp(x.unflatten(-1, (-1, 32)), (scale.int() - 127)[..., None]).flatten(-2)


def _turned(x, positions, inv_freq):
    """Rows (T, heads, hd) with their first features rotated, fp32; angles in 64 bits."""
    half = inv_freq.numel()
    angle = positions.double()[:, None, None] * inv_freq.double()
    c, s = angle.cos().float(), angle.sin().float()
    x = x.float()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def _plain_append(s):
    kp, vp, ks, vs = s["cache"]
    page, fmt = kp.shape[2], s["case"]["fmt"]
    q = _turned(s["q"], s["positions"], s["inv_freq"]).to(s["q"].dtype)
    k, v = _turned(s["k"], s["positions"], s["inv_freq"]), s["v"].float()
    at, off = s["table"][s["rows"].long(), s["positions"].long() // page].long(), s["positions"].long() % page
    if ks is None:
        kp[at, :, off], vp[at, :, off] = k.to(kp.dtype), v.to(vp.dtype)
    else:
        (kp[at, :, off], ks[at, :, off]), (vp[at, :, off], vs[at, :, off]) = _quantize(k, fmt), _quantize(v, fmt)
    if "cu" not in s:
        return (q, *_cache_values(s["cache"]))
    t = torch.arange(s["total"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long().contiguous(), t, right=True)
    pos = t - s["cu"].long()[seq]
    at, off = s["table"][seq, pos // page].long(), pos % page
    return q, *(_values(x[at, :, off], None if y is None else y[at, :, off]).to(torch.bfloat16)
                for x, y in ((kp, ks), (vp, vs)))


def _cache_values(cache):
    """The cache itself; e4m3 codes as the numbers they stand for."""
    k, v, ks, vs = cache
    return (k, v) if ks is None else (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs)


def _plain_pages(pages, scale, table):
    """The table's pages as (B, Hkv, tokens, hd) fp32."""
    at = table.long().clamp(min=0)
    x = _values(pages[at], None if scale is None else scale[at])
    B, P, Hkv, page, hd = x.shape
    return x.transpose(1, 2).reshape(B, Hkv, P * page, hd)


def _plain_attend(s):
    q, (kp, vp, ks, vs) = s["q"], s["cache"]
    B, H, hd = q.shape[0], q.shape[-2], q.shape[-1]
    k = _plain_pages(kp, ks, s["table"])
    Hkv, tokens = k.shape[1], k.shape[2]
    x = q.view(B, -1, Hkv, H // Hkv, hd).float().transpose(1, 2)
    N, G = x.shape[2:4]
    w = (x.reshape(B, Hkv, N * G, hd) @ k.transpose(-1, -2).contiguous()).mul_(s["scale"]).view(B, Hkv, N, G, tokens)
    del k
    live = torch.full_like(s["lens"], N) if s["live"] is None else s["live"]
    i, j = torch.arange(N, device=DEV)[None, :, None], torch.arange(tokens, device=DEV)[None, None]
    seen = (j < (s["lens"] - live + 1)[:, None, None] + i) & (i < live[:, None, None])
    w.masked_fill_(~seen[:, None, :, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    w.div_(w.sum(-1, keepdim=True).clamp(min=1e-38))
    o = w.view(B, Hkv, N * G, tokens) @ _plain_pages(vp, vs, s["table"])
    return o.view(B, Hkv, N, G, hd).transpose(1, 2).reshape(q.shape).to(q.dtype)


def _plain_verify(s):
    x, drafts, q, n = s["logits"].double(), s["drafts"], s["draft_probs"], s["draft_lens"].long()
    B, N, V = x.shape[0], x.shape[1] - 1, x.shape[2]
    t = s["temperature"].double()[:, None, None]
    top = x.amax(-1, keepdim=True)
    cols = torch.arange(V, device=DEV)
    first = torch.where(x == top, cols, V).amin(-1, keepdim=True)
    p = ((x - top) / torch.where(t > 0, t, 1.0)).exp_()
    p = torch.where(t > 0, p.div_(p.sum(-1, keepdim=True)), (cols == first).double())
    at = drafts.long()[..., None]
    qx = torch.ones_like(drafts, dtype=torch.float64) if q is None else q.gather(2, at)[..., 0].double()
    ok = (s["uniforms"][:, :N].double() * qx < p[:, :N].gather(2, at)[..., 0]) & (torch.arange(N, device=DEV) < n[:, None])
    accepted = ok.long().cumprod(-1).sum(-1)
    b = torch.arange(B, device=DEV)
    p = p[b, accepted]
    if N:
        turned = (accepted < n)[:, None]
        i = accepted.clamp(max=N - 1)
        less = (cols == drafts.long()[b, i][:, None]).double() if q is None else q[b, i].double()
        w = (p - less).clamp_(min=0.0)
        p = torch.where(turned & (w.sum(-1, keepdim=True) > 0), w, p)
    c = p.cumsum(-1)
    token = (c <= s["uniforms"][:, N:].double() * c[:, -1:]).sum(-1).minimum(torch.where(p > 0, cols, 0).amax(-1))
    i = torch.arange(N + 1, device=DEV)[None]
    given = torch.cat([drafts.long(), drafts.new_zeros(B, 1, dtype=torch.long)], 1)
    tokens = torch.where(i < accepted[:, None], given, torch.where(i == accepted[:, None], token[:, None], -1))
    return tokens, accepted.to(torch.int32)


def _plain(s):
    return {"append": _plain_append, "extend": _plain_append, "attend": _plain_attend,
            "verify": _plain_verify}[s["case"]["kind"]](s)


# ---- the package's entry points ------------------------------------------------


def _own(s):
    from naylis_amd import mom_kernels as mk
    kind = s["case"]["kind"]
    if kind in ("append", "extend"):
        cache = mk.PagedCache(*s["cache"])
        q = mk.paged_append_rope(cache, s["q"], s["k"], s["v"], s["inv_freq"], s["table"], s["positions"], s["rows"])
        if kind == "append":
            return (q, *_cache_values(s["cache"]))
        return (q, *mk.paged_gather(cache, s["table"], s["cu"], s["total"]))
    if kind == "attend":
        return mk.paged_attention(s["q"], mk.PagedCache(*s["cache"]), s["table"], s["lens"], scale=s["scale"],
                                  q_lens=s["live"])
    return tuple(mk.verify_drafts(s["logits"], s["drafts"], s["uniforms"], draft_probs=s["draft_probs"],
                                  draft_lens=s["draft_lens"], temperature=s["temperature"]))


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- work --------------------------------------------------------------------


def _row(case):
    """Bytes of a token's key (or value) in the cache, all heads."""
    return case["Hkv"] * {"bf16": 2 * case["hd"], "e4m3": case["hd"] + 4, "e2m1": case["hd"] // 2 + case["hd"] // 32}[case["fmt"]]


def work(case):
    kind = case["kind"]
    if kind in ("append", "extend"):
        given = case["T"] * (2 * case["H"] + 2 * case["Hkv"]) * case["hd"] * 2 + 2 * case["T"] * _row(case)
        if kind == "append":
            return {"bytes": given, "flops": 0}
        return {"bytes": given + 2 * sum(_ends(case)) * (_row(case) + case["Hkv"] * case["hd"] * 2), "flops": 0}
    if kind == "attend":
        tokens, q = sum(_cache_lens(case)), case["B"] * case["N"] * case["H"] * case["hd"]
        return {"bytes": 2 * tokens * _row(case) + 4 * q, "flops": 4 * tokens * case["N"] * case["H"] * case["hd"]}
    rows = sum(_live(case)) + case["B"]
    drafts = {"none": 0, "f32": 4, "bf16": 2}[case["probs"]] * case["B"] * (case["N"] > 0)  # a row of each sequence
    return {"bytes": case["V"] * (rows * (2 if case["dtype"] == "bf16" else 4) + drafts), "flops": 4 * rows * case["V"]}


# ---- fp64 statements -----------------------------------------------------------


def _rounded(x, bits, lowest):
    """x at `bits` binary digits, fewer below 2^lowest, ties to the even one."""
    step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** lowest))) - (bits - 1))
    return torch.round(x / step) * step


def _exact_codes(x, fmt):
    """The values that rows fp64 have in the cache, as a pair (codes, scale where it is one of a row)."""
    if fmt == "bf16":
        return x, None
    if fmt == "e4m3":
        top = x.abs().amax(-1)
        scale = torch.where(top > 0, top / 448, 1.0)
        return _rounded(x / scale[..., None], 4, -6), scale
    y = x.reshape(*x.shape[:-1], -1, 32)
    top = y.abs().amax(-1, keepdim=True)
    scale = 2.0 ** (torch.floor(torch.log2(top.clamp(min=2.0 ** -124))) - 2)
    return (_rounded(y / scale, 2, 0).clamp(-6, 6) * scale).reshape(x.shape), None


def _exact_turned(x, positions, inv_freq):
    """Pairs of features as complex numbers times e^(i angle)."""
    half = inv_freq.numel()
    x = x.double()
    z = torch.complex(x[..., :half], x[..., half:2 * half])
    angle = positions.double()[:, None] * inv_freq.double()
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_append(s):
    fmt, page = s["case"]["fmt"], s["case"]["page"]
    pos = s["positions"].long()
    slot = s["table"][s["rows"].long(), pos // page].long() * page + pos % page
    res, scales = [], []
    for i, new in enumerate((_exact_turned(s["k"], pos, s["inv_freq"]), s["v"].double())):
        pages, scale = s["cache"][i], s["cache"][i + 2]
        old = pages.view(torch.float8_e4m3fn).double() if fmt == "e4m3" else _values(pages, scale).double()
        old = old.transpose(1, 2).reshape(-1, *new.shape[1:])
        new, new_scale = _exact_codes(new, fmt)
        old[slot] = new
        if fmt == "e4m3":
            at = scale.double().transpose(1, 2).reshape(-1, new.shape[1])
            at[slot] = new_scale
            scales.append(at)
        res.append(old)
    q = _exact_turned(s["q"], pos, s["inv_freq"])
    if s["case"]["kind"] == "append":
        shape = s["cache"][0].shape
        back = lambda x: x.reshape(shape[0], page, *x.shape[1:]).transpose(1, 2)  # noqa: E731
        return (q, *(back(x) for x in res), *(back(x) for x in scales))
    if scales:
        res = [x * y[..., None] for x, y in zip(res, scales)]
    ends = s["cu"].tolist()
    t = torch.cat([s["table"][b].long().repeat_interleave(page)[:n] * page + torch.arange(n, device=DEV) % page
                   for b, n in enumerate(y - x for x, y in zip(ends, ends[1:]))])
    return q, res[0][t], res[1][t]


def _exact_attend(s):
    case, (kp, vp, ks, vs) = s["case"], s["cache"]
    B, N, H, hd, page = case["B"], case["N"], case["H"], case["hd"], case["page"]
    q = s["q"].double().view(B, N, H, hd)
    out = torch.zeros(B, N, H, hd, dtype=torch.float64, device=DEV)
    live = [1] * B if s["live"] is None else _live(case)
    for b, n in enumerate(_cache_lens(case)):
        ids = s["table"][b, :-(-n // page)].long()
        for h in range(H):
            c = h // (H // case["Hkv"])
            k, v = (_values(x[ids, c], None if y is None else y[ids, c]).double().reshape(-1, hd)[:n]
                    for x, y in ((kp, ks), (vp, vs)))
            for i in range(live[b]):
                m = n - (live[b] - 1 - i)
                if m > 0:
                    out[b, i, h] = torch.softmax(k[:m] @ q[b, i, h] * s["scale"], 0) @ v[:m]
    return out.view(s["q"].shape)


def _exact_verify(s):
    case = s["case"]
    N, V = case["N"], case["V"]
    tokens, counts = [], []
    drafts, u = s["drafts"].tolist(), s["uniforms"].tolist()
    for b, n in enumerate(_live(case)):
        t = float(s["temperature"][b])
        less, row = None, []
        for i in range(n + 1):
            x = s["logits"][b, i].double()
            if t > 0:
                p = torch.softmax(x / t, 0)
            else:
                p = torch.zeros(V, dtype=torch.float64, device=DEV)
                p[int((x == x.max()).nonzero()[0])] = 1
            if i == n:
                break
            d = drafts[b][i]
            q = 1.0 if s["draft_probs"] is None else float(s["draft_probs"][b, i, d])
            if u[b][i] * q < float(p[d]):
                row.append(d)
                continue
            less = p.clone()
            if s["draft_probs"] is None:
                less[d] = 0
            else:
                less = (p - s["draft_probs"][b, i].double()).clamp(min=0)
            break
        w = p if less is None or float(less.sum()) == 0 else less
        c = torch.cumsum(w, 0)
        at = int(torch.searchsorted(c, u[b][N] * c[-1], right=True))
        counts.append(len(row))
        row.append(min(at, int(w.nonzero()[-1])))
        tokens.append(row + [-1] * (N + 1 - len(row)))
    return torch.tensor(tokens).to(DEV), torch.tensor(counts, dtype=torch.int32).to(DEV)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend" and sum(_cache_lens(case)) * case["H"] * case["N"] > 6e7 and case["B"] * case["H"] * case["N"] > 6000:
        return None
    return {"append": _exact_append, "extend": _exact_append, "attend": _exact_attend, "verify": _exact_verify}[kind](s)

"""A paged cache of 8-bit keys and values and what keeps it short: what is timed, in plain torch and through
`castforge_amd.ops`.

  append   rotation of queries and keys, and keys and values as E4M3 codes into the pages of a cache, with one scale a
           page and head that grows with its tokens; every cached token of the pages that were written is read back,
           as the values that they stand for
  attend   softmax(scale q K^T) V over that cache: single queries of many sequences, a few, or whole prompts; over all
           tokens up to the query's own, or over a window of the last ones and a few first ones (sinks)
  observe  the same, and the weights that each cached token got, summed over the queries, added to its earlier ones
  evict    the tokens of each sequence and head that have the greatest weights, and the first and the last ones, moved
           to new pages in their order; the new pages are read back

`listed()` holds fixed cases, `draw(rng)` gives further ones of the same ranges:
  1..8 heads of keys with 1..8 query heads each, of 64 or 128 channels; pages of 16..256 tokens; 1..128 sequences of
  1..131072 tokens, at most 600000 together; 1..8192 queries; windows of 16..16384 tokens behind 0..64 sinks.

A page holds [head, token, channel] E4M3 codes and, for each head, one float32 scale: an element stands for code * scale.
"""
import math
import random

import torch

own = False  # True: the framework's entry points; False: elementary torch operations in 32 bits

BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
MOST_PAIRS = 32 * 128 * 8192 * 8192  # query heads x channels x queries x keys of the longest listed prompt, masked ones too
MOST_SEEN = 32 * 128 * 8192 * 1024   # those that are seen
MOST_TOKENS = 600000                 # cached tokens of a pass, all sequences
MOST_CACHED = 32 * 30000 * 8 * 128   # elements of K that a pass may hold


def listed():
    return [
        # a decode batch's new tokens into pages in use: latency
        {"name": "append_b16", "op": "append", "b": 16, "q": 1, "kv": 3000, "hkv": 8, "ratio": 4, "d": 128, "page": 64,
         "ragged": True, "rot": 128, "interleaved": False},
        # a whole prompt's tokens, every head its own keys
        {"name": "append_t4096", "op": "append", "b": 1, "q": 4096, "kv": 4096, "hkv": 32, "ratio": 1, "d": 128, "page": 64,
         "ragged": False, "rot": 128, "interleaved": False},
        # one sequence early in its answer: latency of a short cache
        {"name": "decode_b1", "op": "attend", "b": 1, "q": 1, "kv": 1009, "hkv": 8, "ratio": 4, "d": 128, "page": 64,
         "ragged": False, "window": 0, "sinks": 0},
        # a serving batch of sequences of many lengths
        {"name": "decode_b48", "op": "attend", "b": 48, "q": 1, "kv": 8000, "hkv": 8, "ratio": 4, "d": 128, "page": 16,
         "ragged": True, "window": 0, "sinks": 0},
        # a few guessed tokens of each sequence checked at once, 64-channel heads
        {"name": "verify_b12_q5", "op": "attend", "b": 12, "q": 5, "kv": 3001, "hkv": 8, "ratio": 3, "d": 64, "page": 32,
         "ragged": True, "window": 0, "sinks": 0},
        # a whole prompt
        {"name": "prompt_4096", "op": "attend", "b": 1, "q": 4096, "kv": 4096, "hkv": 8, "ratio": 4, "d": 128, "page": 64,
         "ragged": False, "window": 0, "sinks": 0},
        # long conversations that look back over a window and at their first tokens
        {"name": "window_decode_b32", "op": "attend", "b": 32, "q": 1, "kv": 30000, "hkv": 8, "ratio": 4, "d": 128, "page": 64,
         "ragged": True, "window": 4096, "sinks": 4},
        # a long prompt of a model with a window: the largest attention
        {"name": "window_prompt_8192", "op": "attend", "b": 1, "q": 8192, "kv": 8192, "hkv": 8, "ratio": 4, "d": 128, "page": 64,
         "ragged": False, "window": 1024, "sinks": 4},
        # a decode batch that keeps count of what its tokens are worth
        {"name": "observe_b32", "op": "observe", "b": 32, "q": 1, "kv": 8000, "hkv": 8, "ratio": 4, "d": 128, "page": 64,
         "ragged": True, "window": 0, "sinks": 0},
        # a prompt's last tokens, whose weights decide what the cache keeps of it; an odd number of heads a group
        {"name": "observe_q64", "op": "observe", "b": 1, "q": 64, "kv": 16384, "hkv": 4, "ratio": 7, "d": 128, "page": 128,
         "ragged": False, "window": 0, "sinks": 0},
        # one sequence's cache cut to a quarter: latency
        {"name": "evict_b1", "op": "evict", "b": 1, "kv": 4001, "keep": 1000, "hkv": 8, "d": 128, "page": 16, "ragged": False,
         "first": 4, "last": 64},
        # a batch's caches cut to what a window would hold
        {"name": "evict_b32", "op": "evict", "b": 32, "kv": 8192, "keep": 2048, "hkv": 8, "d": 128, "page": 64, "ragged": True,
         "first": 4, "last": 512},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "attend", "observe", "observe", "evict", "evict"])
    d, hkv, ratio = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    case = {"op": op, "hkv": hkv, "d": d, "page": rng.choice([16, 32, 64, 64, 128, 256]), "ragged": rng.random() < 0.6}
    if op == "evict":
        b = log(1, 64)
        kv = max(2, min(log(64, 131072), 32 * 8192 // b))
        keep = log(1, kv)
        first, last = min(keep, rng.choice([0, 1, 4, 4, 16])), rng.choice([0, 1, log(1, 512)])
        return {**case, "b": b, "kv": kv, "keep": keep, "first": first, "last": min(last, keep - first)}
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    b = log(1, 16 if kind == "prompt" else 128)
    q = 1 if kind == "decode" else rng.randint(2, 16) if kind == "verify" else log(17, 8192)
    kv = q + rng.choice([0, 0, log(1, 16384)]) if kind == "prompt" else max(q, log(1, 131072))
    window = rng.choice([0, 0, log(16, 16384)])
    if op == "append":
        kv, window = min(kv, 16384), 0
        q = min(q, 4096)
    # a pass holds, and compares, no more than the largest listed ones
    heads = hkv * ratio * d * b
    kv = max(1, min(kv, MOST_TOKENS // b, MOST_CACHED // (b * hkv * d)))
    q = max(1, min(q, kv, MOST_PAIRS // (heads * kv), MOST_SEEN // (heads * min(kv, window + 64 if window else kv))))
    case |= {"b": b, "q": q, "kv": kv, "ratio": ratio}
    if op == "append":
        return {**case, "rot": rng.choice([d, d, d // 2]), "interleaved": rng.random() < 0.4}
    return {**case, "window": window, "sinks": rng.choice([0, 1, 4, 4, 64]) if window else 0}


def lengths(case):
    """(queries, cached tokens) of each sequence; ragged ones run from a tenth of the longest to all of it."""
    r, got = random.Random(case["kv"] * 1000 + case["b"]), []
    for i in range(case["b"]):
        f = 1.0 if not case["ragged"] or i == 0 else r.uniform(0.1, 1.0)
        kv, most = max(1, int(case["kv"] * f)), case.get("q", 1)
        q = 1 if most == 1 else max(1, int(most * (f if most > 16 else r.uniform(0.3, 1.0))))
        got.append((min(q, kv), kv))
    return got


# ------------------------------------------------------------------------------ inputs ----
def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000 + part)
    return g


def _pages(pages, hkv, page, d, g):
    """Codes and scales of a cache in use: N(0, 0.2 .. 1.6) by page and head, some channels four times larger."""
    x = torch.randn((pages, hkv, page, d), generator=g, device="cuda") * 52
    big = torch.rand((hkv, 1, d), generator=g, device="cuda") < 0.03
    codes = torch.where(big, x * 4, x).clamp(-448, 448).to(F8).view(torch.uint8)
    return codes, torch.ldexp(torch.ones((), device="cuda"), torch.randint(-8, -4, (pages, hkv), generator=g, device="cuda"))


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    s, g = dict(case), _gen(seed, 0)
    hkv, d, page, b = case["hkv"], case["d"], case["page"], case["b"]
    lens = lengths(case)
    need = [-(-kv // page) for _, kv in lens]
    kept = [min(kv, case.get("keep", 0)) for _, kv in lens]
    new = [-(-n // page) for n in kept]
    pages = sum(need) + sum(new) + 3
    s["cache"] = _pages(pages, hkv, page, d, g) + _pages(pages, hkv, page, d, g)
    at = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)

    def table(counts, first):
        counts = _int(counts, torch.int64)
        begin, col = first + counts.cumsum(0) - counts, torch.arange(int(counts.max()), device="cuda")
        return torch.where(col < counts[:, None], at[(begin[:, None] + col).clamp(max=pages - 1)], 0)

    s["table"], s["spare"] = table(need, 0), at[-1]
    s["kv_lens"] = _int([kv for _, kv in lens])
    s["longest"] = max(kv for _, kv in lens)
    if case["op"] == "evict":
        s["new_table"] = table(new, sum(need))
        # what attention gave each token: a few have most of it, many have had none
        w = torch.exp(2 * torch.randn((b, hkv, s["table"].shape[1] * page), generator=g, device="cuda"))
        s["weights"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.2, 0.0, w)
        row = torch.repeat_interleave(torch.arange(b, device="cuda"), _int(kept, torch.int64))
        place = torch.cat([torch.arange(n, device="cuda") for n in kept])
        s["slots"] = s["new_table"][row, place // page].long() * page + place % page
        return s
    hq, n = hkv * case["ratio"], sum(q for q, _ in lens)
    s["cu_q"] = _int([sum(q for q, _ in lens[:i]) for i in range(b + 1)])
    s["longest_q"] = max(q for q, _ in lens)
    if case["op"] == "append":
        half = case["rot"] // 2
        # one projection's output: the rows of q, k and v lie behind one another
        qkv = torch.randn((n, (hq + 2 * hkv) * d), generator=g, device="cuda")
        big = torch.rand((hq + 2 * hkv) * d, generator=g, device="cuda") < 0.03
        qkv = torch.where(big, qkv * 6, qkv).to(BF16).unflatten(1, (-1, d))
        s["qs"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["positions"] = torch.cat([torch.arange(kv - q, kv, device="cuda") for q, kv in lens])
        angle = torch.arange(case["kv"], device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        s["cos"], s["sin"] = angle.cos(), angle.sin()
        # the cached tokens of the pages that get new ones, and those pages
        first = [(kv - q) // page * page for q, kv in lens]
        row = torch.repeat_interleave(torch.arange(b, device="cuda"), _int([kv - f for (_, kv), f in zip(lens, first)], torch.int64))
        place = torch.cat([torch.arange(f, kv, device="cuda") for (_, kv), f in zip(lens, first)])
        s["slots"] = s["table"][row, place // page].long() * page + place % page
        s["touched"] = torch.unique(s["slots"] // page)
        return s
    s["qs"] = (1.5 * torch.randn((n, hq, d), generator=g, device="cuda")).to(BF16)
    if case["op"] == "observe":
        # of as many queries before as there are now
        s["weights"] = torch.rand((b, hkv, s["table"].shape[1] * page), generator=g, device="cuda") * (2 * case["q"] * case["ratio"] / case["kv"])
    return s


# ----------------------------------------------------------------------- the framework ----
def _run_own(s):
    from castforge_amd import ops

    op, cache = s["op"], ops.Kv8Cache(*s["cache"])
    if op == "evict":
        kept, lens, weights = ops.kv8_evict(cache, s["table"], s["kv_lens"], s["weights"], s["keep"], s["new_table"], sinks=s["first"],
                                            recent=s["last"])
        return (kept, lens, weights) + ops.kv8_gather(cache, s["slots"])
    cu_q = None if s["q"] == 1 else s["cu_q"]
    if op == "append":
        q = ops.kv8_append(cache, s["k"], s["v"], s["table"], s["kv_lens"], cu_q=cu_q, positions=s["positions"], cos=s["cos"], sin=s["sin"],
                           q=s["qs"], interleaved=s["interleaved"])
        return (q,) + ops.kv8_gather(cache, s["slots"])
    if op == "attend":
        return ops.kv8_attention(s["qs"], cache, s["table"], s["kv_lens"], cu_q=cu_q, window=s["window"] or None, sinks=s["sinks"])
    weights = s["weights"].clone()
    o = ops.kv8_attention(s["qs"], cache, s["table"], s["kv_lens"], cu_q=cu_q, window=s["window"] or None, sinks=s["sinks"], weights=weights)
    return o, weights


# ------------------------------------------------------------------------- plain torch ----
def _rotate(x, cos, sin, rot, interleaved):
    """x [T, H, D] f32: its first `rot` channels turned in pairs (i, i + rot / 2), or (2 i, 2 i + 1)."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = cos[:, None], sin[:, None]
    u, v = a * c - b * s, b * c + a * s
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _power(amax):
    """The least power of two that brings amax to 448 or less, from 2^-70 to 2^30."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875)).clamp(-70, 30))


def _store(codes, scales, x, pages, places, touched):
    """x [T, H, D] f32 into (page, place) of each token; what the touched pages held goes over to their new scale."""
    amax = torch.zeros_like(scales).index_reduce_(0, pages, x.abs().amax(-1), "amax", include_self=True)[touched]
    fresh = torch.zeros(scales.shape[0], dtype=torch.int32, device="cuda").index_reduce_(0, pages, (places == 0).int(), "amax")[touched]
    old = torch.where(fresh[:, None] > 0, 0.0, scales[touched])
    scales[touched] = torch.maximum(old, _power(amax))
    held = codes[touched].view(F8).float() * (old / scales[touched])[..., None, None]
    codes[touched] = held.to(F8).view(torch.uint8)
    codes[pages, :, places] = (x / scales[pages][..., None]).to(F8).view(torch.uint8)


def _rows(cache, slots, page):
    """Keys and values of the slots, [T, H, D]: exact in 16 bits."""
    kc, ks, vc, vs = cache
    p, o = slots // page, slots % page
    return tuple((c[p, :, o].view(F8).float() * t[p][..., None]).to(BF16) for c, t in ((kc, ks), (vc, vs)))


def _evict(s):
    kc, ks, vc, vs = s["cache"]
    page, keep, (b, hkv, length) = s["page"], s["keep"], s["weights"].shape
    lens, table, new = s["kv_lens"].long()[:, None], s["table"].long(), s["new_table"].long()
    t = torch.arange(length, device="cuda")
    kept = (t < s["first"]) | (t >= lens - s["last"])
    rank = torch.where(kept[:, None], math.inf, s["weights"]).masked_fill((t >= lens)[:, None], -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    i = torch.arange(keep, device="cuda")
    best = torch.where(i < lens[:, None], best, length).sort(-1).values
    live, at = best < length, best.clamp(max=length - 1)
    p, h = table.gather(1, (at // page).flatten(1)).view(at.shape), torch.arange(hkv, device="cuda")[:, None]
    # past a sequence's last page: into one that nobody has
    to = torch.where(i // page * page < lens, new[:, i // page], s["spare"])[:, None].expand(-1, hkv, -1)
    for codes, scales in ((kc, ks), (vc, vs)):
        x = codes[p, h, at % page].view(F8).float()
        f = torch.where(live, scales[p, h], 0.0)
        tops = torch.nn.functional.pad(f, (0, -keep % page)).unflatten(-1, (-1, page)).amax(-1)
        top = tops[..., i // page]
        scales[to, h] = top
        codes[to, h, i % page] = (x * (f / top.clamp(min=2.0**-120))[..., None]).to(F8).view(torch.uint8)
    weights = torch.where(live, s["weights"].gather(2, at), 0.0)
    return (torch.where(live, best, -1).int(), lens[:, 0].clamp(max=keep).int(), weights) + _rows(s["cache"], s["slots"], page)


def run(s):
    if own:
        return _run_own(s)
    op, page = s["op"], s["page"]
    if op == "evict":
        return _evict(s)
    kc, ks, vc, vs = s["cache"]
    table, cu, lens, nq = s["table"].long(), s["cu_q"].long(), s["kv_lens"].long()[:, None], s["longest_q"]
    count = (cu[1:] - cu[:-1])[:, None]
    token = torch.arange(s["qs"].shape[0], device="cuda")
    seq = torch.searchsorted(cu, token, right=True) - 1
    if op == "append":
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        q = _rotate(s["qs"].float(), cos, sin, s["rot"], s["interleaved"]).to(BF16)
        at = (lens - count)[seq, 0] + token - cu[seq]
        pages, places = table[seq, at // page], at % page
        _store(kc, ks, _rotate(s["k"].float(), cos, sin, s["rot"], s["interleaved"]), pages, places, s["touched"])
        _store(vc, vs, s["v"].float(), pages, places, s["touched"])
        return (q,) + _rows(s["cache"], s["slots"], page)
    # the tokens that some query of a sequence sees, padded to the longest: the first ones, and the window's
    window = s["window"] or s["longest"]
    span = min(s["longest"], s["sinks"] + window + nq - 1)
    j = torch.arange(span, device="cuda")
    tok = torch.where(j < s["sinks"], j, (lens - span).clamp(min=0) + j)
    near = tok.clamp(max=s["longest"] - 1)
    p, o = table.gather(1, near // page), near % page
    k, v = ((c[p, :, o].view(F8).float() * t[p][..., None]).transpose(1, 2) for c, t in ((kc, ks), (vc, vs)))
    b, hkv, _, d = k.shape
    ratio = s["ratio"]
    at = cu[:-1, None] + torch.arange(nq, device="cuda")
    q = s["qs"][at.clamp(max=s["qs"].shape[0] - 1)].float().view(b, nq, hkv, ratio, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = ((q @ k.transpose(2, 3)) / math.sqrt(d)).view(b, hkv, ratio, nq, span)
    # query i of n sees the keys up to its own place, counted from the end: the window's last ones and the first of all
    mine = (lens - count + torch.arange(nq, device="cuda"))[..., None]
    seen = (tok[:, None] <= mine) & ((tok[:, None] > mine - window) | (tok[:, None] < s["sinks"])) & (torch.arange(nq, device="cuda") < count)[..., None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    w = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (w.view(b, hkv, ratio * nq, span) @ v).view(b, hkv, ratio, nq, d)[seq, :, :, token - cu[seq]].flatten(1, 2).to(BF16)
    if op == "attend":
        return o
    return o, s["weights"].scatter_add(2, near[:, None].expand(-1, hkv, -1), w.sum((2, 3)))


# ------------------------------------------------------------------------------- bounds ----
def work(case):
    d, hkv, page, lens = case["d"], case["hkv"], case["page"], lengths(case)
    if case["op"] == "evict":
        kept = sum(min(kv, case["keep"]) for _, kv in lens)
        # weights in; index and weight out; codes in, out and read back; given out in 16 bits
        return {"bytes": hkv * (4 * sum(kv for _, kv in lens) + kept * (8 + 6 * d + 4 * d)), "flops": sum(kv for _, kv in lens) * hkv + 2 * kept * hkv * d}
    hq, n = hkv * case["ratio"], sum(q for q, _ in lens)
    if case["op"] == "append":
        read = sum(kv - (kv - q) // page * page for q, kv in lens)
        # q in and out, k and v in, as codes out; the table's rows and positions; the pages read back and given out in 16 bits
        return {"bytes": n * (4 * hq * d + 4 * hkv * d + 2 * hkv * d + 4 * case["rot"] + 8) + read * hkv * d * (2 + 4), "flops": n * (6 * (hq + hkv) * case["rot"] + 4 * hkv * d)}
    window, sinks, pairs, spans = case["window"] or case["kv"], case["sinks"], 0, 0
    for q, kv in lens:
        spans += min(kv, sinks + window + q - 1)
        # query at place p sees min(p + 1, sinks + window) tokens
        whole = min(kv, max(kv - q, sinks + window - 1))  # places below see every token up to theirs
        pairs += (whole * (whole + 1) - (kv - q) * (kv - q + 1)) // 2 + (kv - whole) * (sinks + window)
    more = 8 * hkv * spans if case["op"] == "observe" else 0
    return {"bytes": 4 * n * hq * d + 2 * spans * hkv * d + more, "flops": 4 * hq * d * pairs}


# ------------------------------------------------------------------------------ 64 bits ----
def exact(case, seed):
    """What `run` returns, in float64; what is held in 8 bits, as the values that it stands for."""
    s = prepare(case, seed)
    hkv, d, page, lens = case["hkv"], case["d"], case["page"], lengths(case)
    kc, ks, vc, vs = s["cache"]

    def held(codes, scales, i, tokens):
        """The values of sequence i's tokens, [H, tokens, D]."""
        ids = s["table"][i, tokens // page].long()
        return (codes[ids, :, tokens % page].view(F8).double() * scales[ids].double()[..., None]).transpose(0, 1)

    def rounded(x, scale):
        return (x / scale).to(F8).double() * scale

    def power(amax):
        return 2.0 ** math.ceil(math.log2(amax / 448)) if amax else 2.0**-70

    if case["op"] == "evict":
        index, weights, ks_out, vs_out = [], [], [], []
        for i, (_, kv) in enumerate(lens):
            n, rows = min(kv, case["keep"]), ([], [])
            for h in range(hkv):
                w = s["weights"][i, h, :kv].double().cpu().numpy().tolist()
                always = set(range(min(case["first"], kv))) | set(range(max(0, kv - case["last"]), kv))
                rest = sorted((t for t in range(kv) if t not in always), key=lambda t: (-w[t], t))
                chosen = sorted(sorted(always) + rest[:n - len(always)]) if n > len(always) else sorted(always)[:n]
                index.append(chosen + [-1] * (case["keep"] - n))
                weights.append([w[t] for t in chosen] + [0.0] * (case["keep"] - n))
                tokens = torch.tensor(chosen, device="cuda")
                for got, (c, f) in zip(rows, ((kc, ks), (vc, vs))):
                    ids = s["table"][i, tokens // page].long()
                    parts = [(x * g[:, None] / g.max()).to(F8).double() * g.max() for x, g in
                             zip(c[ids, h, tokens % page].view(F8).double().split(page), f[ids, h].double().split(page))]
                    got.append(torch.cat(parts))
            ks_out.append(torch.stack(rows[0], 1))
            vs_out.append(torch.stack(rows[1], 1))
        shape = (case["b"], hkv, case["keep"])
        return (torch.tensor(index).view(shape).int(), torch.tensor([min(kv, case["keep"]) for _, kv in lens]).int(),
                torch.tensor(weights, dtype=torch.float64).view(shape), torch.cat(ks_out), torch.cat(vs_out))
    if case["op"] == "append":
        n = case["rot"]
        half = n // 2
        c, t = s["cos"].double()[s["positions"]][:, None], s["sin"].double()[s["positions"]][:, None]

        def turn(x):
            x = x.double().clone()
            one, two = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, half), slice(half, n))
            a, b = x[..., one].clone(), x[..., two].clone()
            x[..., one], x[..., two] = a * c - b * t, a * t + b * c
            return x

        out, first = [[], []], 0
        rows = (turn(s["k"]), s["v"].double())
        for i, (q, kv) in enumerate(lens):
            for got, x, codes, scales in zip(out, rows, (kc, vc), (ks, vs)):
                for start in range((kv - q) // page * page, kv, page):
                    before, end = max(0, kv - q - start), min(kv, start + page)
                    new = x[first + max(0, start - (kv - q)):first + end - (kv - q)]
                    scale = torch.tensor([power(a) for a in new.abs().amax((0, 2)).tolist()], dtype=torch.float64, device="cuda")
                    if before:
                        old = held(codes, scales, i, torch.arange(start, start + before, device="cuda")).transpose(0, 1)
                        scale = torch.maximum(scale, scales[s["table"][i, start // page].long()].double())
                        got.append(rounded(old, scale[:, None]))
                    got.append(rounded(new, scale[:, None]))
            first += q
        return turn(s["qs"]), torch.cat(out[0]), torch.cat(out[1])
    out, sums, first = [], s["weights"].double() if case["op"] == "observe" else None, 0
    for i, (nq, kv) in enumerate(lens):
        tokens = torch.arange(kv, device="cuda")
        k, v = held(kc, ks, i, tokens), held(vc, vs, i, tokens)
        q = s["qs"][first:first + nq].double()
        place = torch.arange(kv - nq, kv, device="cuda")[:, None]
        hidden = tokens > place
        if case["window"]:
            hidden |= (tokens <= place - case["window"]) & (tokens >= case["sinks"])
        heads = []
        for h in range(q.shape[1]):
            at = h // case["ratio"]
            w = torch.softmax((q[:, h] @ k[at].t() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            heads.append(w @ v[at])
            if sums is not None:
                sums[i, at, :kv] += w.sum(0)
        out.append(torch.stack(heads, 1))
        first += nq
    return torch.cat(out) if sums is None else (torch.cat(out), sums)

"""A paged KV cache held in 8 bits, and attention over a prefix that sequences share, as measured cases.

A quantised cache is two page arrays [n_pages, n_kv_heads, page_tokens, D + D / 32] of 1-byte
values (float8_e4m3fn or int8).  Of each page and head the first page_tokens * D bytes are the
tokens' codes, the rest a scale byte s for every 32 values of a token: a value is code * 2^(s - 127).

  append   RMS norm, rotation and quantised store of new tokens, then the stored rows read back
  read     tokens of a quantised cache as 16-bit rows
  attend   attention of ragged chunks of new tokens over a quantised cache
  prefix   the same for groups of sequences that share their first tokens, whose keys are gone
           through once for a whole group, over a 16-bit or a quantised cache

`run` computes them in elementary torch operations, or (own) by the calls a user makes.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
GROUP = 32                                   # values that share a scale
LARGEST = {"e4m3": 448.0, "int8": 127.0}     # of a code
LOWEST = {"e4m3": -15, "int8": -22}          # exponents of a scale
HIGHEST = 7


# ------------------------------------------------------------------ cases


def listed():
    return [
        # the step before the attention of a decoding batch
        {"name": "append decode batch", "op": "append", "type": "bf16", "cache": "e4m3", "seqs": 64, "new": 1, "kv": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "rotary": 128, "interleaved": False, "norm": True},
        # the chunks of two prompts, half of each head turned in neighbouring pairs
        {"name": "append prompt", "op": "append", "type": "fp16", "cache": "int8", "seqs": 2, "new": 4099, "kv": 5000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "rotary": 64, "interleaved": True, "norm": True},
        # one short conversation taken out of the cache: all latency
        {"name": "read one sequence", "op": "read", "type": "bf16", "cache": "int8", "seqs": 1, "kv": 777, "kv_heads": 8, "dim": 128, "page": 16},
        # a batch of them, for a step that wants 16-bit rows
        {"name": "read batch", "op": "read", "type": "fp16", "cache": "e4m3", "seqs": 16, "kv": 8192, "kv_heads": 8, "dim": 128, "page": 16},
        # one conversation decoding one token: all latency
        {"name": "attend one token", "op": "attend", "type": "bf16", "cache": "e4m3", "seqs": 1, "new": 1, "kv": 777, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": False},
        # a decoding batch of ragged long contexts: bound by reading the cache
        {"name": "attend decode batch", "op": "attend", "type": "bf16", "cache": "e4m3", "seqs": 64, "new": 1, "kv": 16384, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": False},
        # verifying drafted tokens, seven query heads to a key head
        {"name": "attend drafted", "op": "attend", "type": "fp16", "cache": "int8", "seqs": 16, "new": 5, "kv": 5001, "ragged": True, "heads": 28,
         "kv_heads": 4, "dim": 128, "page": 32, "window": 0, "sinks": 0, "lse": True},
        # streaming sequences: a step that mixes a chunk with decoding, a window beside the first tokens
        {"name": "attend window", "op": "attend", "type": "fp16", "cache": "e4m3", "seqs": 8, "new": 1001, "kv": 16000, "ragged": True, "heads": 16,
         "kv_heads": 16, "dim": 64, "page": 64, "window": 1024, "sinks": 4, "lse": False},
        # a whole long prompt: bound by the matrix products
        {"name": "attend prompt", "op": "attend", "type": "bf16", "cache": "int8", "seqs": 1, "new": 8192, "kv": 8192, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": True},
        # four samples of one conversation
        {"name": "prefix samples", "op": "prefix", "type": "bf16", "cache": "16", "groups": 1, "seqs": 4, "new": 1, "prefix": 1001, "tail": 100, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "lse": False},
        # a decoding batch behind one long system prompt
        {"name": "prefix decode batch", "op": "prefix", "type": "bf16", "cache": "16", "groups": 1, "seqs": 64, "new": 1, "prefix": 16384, "tail": 1000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "lse": False},
        # drafted tokens of conversations over a few long documents, held in 8 bits
        {"name": "prefix documents", "op": "prefix", "type": "fp16", "cache": "e4m3", "groups": 3, "seqs": 16, "new": 4, "prefix": 10007, "tail": 500,
         "heads": 28, "kv_heads": 4, "dim": 128, "page": 32, "lse": True},
    ]


def spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def page_for(rng, dim):
    """A page size whose scale bytes are a multiple of 16."""
    return rng.choice([p for p in (8, 16, 16, 24, 32, 48, 64, 128) if p * (dim // GROUP) % 16 == 0])


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "prefix", "prefix", "append", "append", "read"])
    dim = rng.choice([64, 64, 96, 128, 128, 128, 256])
    c = {"op": op, "type": rng.choice(["bf16", "fp16"]), "cache": rng.choice(["e4m3", "int8"]), "dim": dim, "page": page_for(rng, dim),
         "kv_heads": rng.choice([1, 2, 4, 8])}
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "attend":
        c |= {"seqs": spread(rng, 1, 64), "new": spread(rng, 1, 4096), "ragged": rng.random() < 0.7, "window": 0, "sinks": 0, "lse": rng.random() < 0.5}
        c["kv"] = c["new"] + spread(rng, 1, 16384) - 1
        if rng.random() < 0.3:
            c["window"], c["sinks"] = spread(rng, 16, 4096), rng.choice([0, 1, 4, 33])
        while c["seqs"] * c["new"] * c["heads"] * c["kv"] > 1 << 30 or c["seqs"] * c["kv_heads"] * c["kv"] * dim > 1 << 30:
            if c["seqs"] > 1:
                c["seqs"] = c["seqs"] // 2
            else:
                c["new"], c["kv"] = (c["new"] + 1) // 2, c["kv"] // 2 + 1
        return c
    if op == "prefix":
        c |= {"cache": rng.choice(["16", "16", "e4m3", "int8"]), "groups": rng.choice([1, 1, 2, 3, 5]), "seqs": spread(rng, 2, 64), "new": rng.choice([1, 1, 1, 2, 5]),
              "prefix": spread(rng, 64, 16384), "lse": rng.random() < 0.5}
        c["tail"] = c["new"] + spread(rng, 1, 1024)
        while c["groups"] * c["seqs"] * c["kv_heads"] * dim * (c["prefix"] + c["tail"]) > 1 << 31:
            c["seqs"], c["prefix"] = max(2, c["seqs"] // 2), max(64, c["prefix"] // 2)
        return c
    if op == "append":
        c |= {"seqs": spread(rng, 1, 128), "new": spread(rng, 1, 4096), "rotary": rng.choice([dim, dim, dim // 2, 20]), "interleaved": rng.random() < 0.3,
              "norm": rng.random() < 0.7}
        while c["seqs"] * c["new"] > 8192:
            c["seqs"], c["new"] = (c["seqs"] + 1) // 2, (c["new"] + 1) // 2
        c["kv"] = c["new"] + spread(rng, 1, 2048) - 1
        return c
    del c["heads"]
    c |= {"seqs": spread(rng, 1, 64), "kv": spread(rng, 1, 16384)}
    while c["seqs"] * c["kv"] * c["kv_heads"] * dim > 1 << 27:
        c["seqs"], c["kv"] = (c["seqs"] + 1) // 2, (c["kv"] + 1) // 2
    return c


def lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence: a part of the case, not of the seed."""
    r = random.Random(case["seqs"] * 7919 + case["kv"])
    new, kv = [], []
    for i in range(case["seqs"]):
        n = case["new"]
        if case["ragged"] and n > 8 and i > 0:
            n = 1 if i % 2 else max(1, int(n * r.uniform(0.0, 0.25)))  # a chunk beside decoding sequences and short prompts
        k = case["kv"] if i == 0 or not case["ragged"] else int(case["kv"] * r.uniform(0.05, 1.0))
        new.append(n)
        kv.append(max(n, k))
    return new, kv


def read_lengths(case):
    r = random.Random(case["seqs"] * 7919 + case["kv"])
    return [case["kv"] if i == 0 else max(1, int(case["kv"] * r.uniform(0.2, 1.0))) for i in range(case["seqs"])]


def prefix_lengths(case):
    """(prefix of each group, cached tokens of each sequence): sequences lie group by group."""
    r = random.Random(case["seqs"] * 7919 + case["prefix"])
    prefix = [case["prefix"] if g == 0 else max(1, int(case["prefix"] * r.uniform(0.3, 1.0))) for g in range(case["groups"])]
    return prefix, [p + max(case["new"], int(case["tail"] * r.uniform(0.05, 1.0))) for p in prefix for _ in range(case["seqs"])]


# ------------------------------------------------------------------ inputs


def normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def packed(lens):
    return ints([0] + lens).cumsum(0).to(torch.int32)


def parts(pages):
    """The codes [n, heads, page_tokens, D] and scale bytes [n, heads, page_tokens, D / 32] of a quantised page array: views."""
    n, h, t, row = pages.shape
    groups = row // (GROUP + 1)
    flat = pages.view(torch.uint8).reshape(n, h, t * row)
    return flat[..., : t * groups * GROUP].unflatten(-1, (t, groups * GROUP)), flat[..., t * groups * GROUP:].unflatten(-1, (t, groups))


def quantised(x, kind):
    """(codes, scale bytes) of fp32 or fp64 x [..., D] as uint8: the smallest scale that holds the group's largest value."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    m, k = torch.frexp(top)
    limit, power = math.frexp(LARGEST[kind])
    e = torch.where(top == 0, LOWEST[kind], k - power + (m > limit)).clamp(LOWEST[kind], HIGHEST)
    y = torch.ldexp(g, -e[..., None]).clamp(-LARGEST[kind], LARGEST[kind]).flatten(-2)
    codes = y.float().to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().to(torch.int8)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def values(codes, scales, kind):
    """What they stand for, in fp32 (exact)."""
    v = codes.contiguous().view(CODES[kind]).float()
    s = (scales.to(torch.int32) << 23).view(torch.float32)
    return (v.unflatten(-1, (-1, GROUP)) * s[..., None]).flatten(-2)


def cache_of(case, g, n_pages):
    """Two page arrays; quantised ones of normal values whose size changes along the head, a few dimensions being large."""
    h, t, d, kind = case["kv_heads"], case["page"], case["dim"], case["cache"]
    if kind == "16":
        return normal(g, (n_pages, h, t, d), DTYPES[case["type"]]), normal(g, (n_pages, h, t, d), DTYPES[case["type"]])
    sizes = torch.exp(0.5 * torch.randn((2, h, 1, d), generator=g, device="cuda"))
    sizes = sizes / sizes.square().mean(-1, keepdim=True).sqrt()
    made = []
    for i in range(2):
        pages = torch.empty((n_pages, h, t, d + d // GROUP), dtype=torch.uint8, device="cuda")
        codes, scales = parts(pages)
        step = max(1, (1 << 27) // (h * t * d))
        for a in range(0, n_pages, step):
            b = min(n_pages, a + step)
            codes[a:b], scales[a:b] = quantised(normal(g, (b - a, h, t, d), torch.float32) * sizes[i], kind)
        made.append(pages.view(CODES[kind]))
    return made


def scattered(g, n_pages, counts, width):
    """A page table whose rows hold `counts` pages each, taken from shuffled pages; -1 behind them."""
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([0] + counts[:-1], device="cuda").cumsum(0)
    at = torch.arange(width, device="cuda")[None, :]
    held = at < torch.tensor(counts, device="cuda")[:, None]
    return torch.where(held, perm[(first[:, None] + at).clamp(max=n_pages - 1)], -1).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"append": prepare_append, "read": prepare_read, "attend": prepare_attend, "prefix": prepare_prefix}[case["op"]](case, g)
    return s | {"case": case, "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def prepare_append(case, g):
    new, kv = lengths(dict(case, ragged=False))
    page, dtype, half = case["page"], DTYPES[case["type"]], case["rotary"] // 2
    counts = [-(-k // page) for k in kv]
    # only the pages that the new tokens lie on are in the cache here, the table's earlier entries point at them too
    tail = [min(c, -(-n // page) + 1) for c, n in zip(counts, new)]
    n_pages = sum(tail) + 3
    k_pages, v_pages = cache_of(case, g, n_pages)
    last = scattered(g, n_pages, tail, max(tail))
    at = torch.arange(max(counts), device="cuda")[None, :] - (ints(counts) - ints(tail))[:, None]
    table = torch.gather(last, 1, at.clamp(0, max(tail) - 1).long()).to(torch.int32).contiguous()
    total, hq, hk, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    turn = torch.arange(max(kv), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)[None, :]
    weight = [(1 + 0.1 * normal(g, (d,), torch.float32)).to(dtype) if case["norm"] else None for _ in range(2)]
    return {"qkv": normal(g, (total, hq + 2 * hk, d), dtype, 2.0),  # the output of one projection
            "k_pages": k_pages, "v_pages": v_pages, "table": table, "cu": packed(new), "kv_len": ints(kv),
            "rope": torch.stack([turn.cos(), turn.sin()], -1).float().contiguous(), "q_weight": weight[0], "k_weight": weight[1],
            "out": torch.empty((total, hq, d), dtype=dtype, device="cuda")}


def prepare_read(case, g):
    kv = read_lengths(case)
    counts = [-(-k // case["page"]) for k in kv]
    n_pages = sum(counts) + 5
    k_pages, v_pages = cache_of(case, g, n_pages)
    return {"k_pages": k_pages, "v_pages": v_pages, "table": scattered(g, n_pages, counts, max(counts)), "cu": packed(kv), "kv_len": ints(kv), "rows": sum(kv)}


def prepare_attend(case, g):
    new, kv = lengths(case)
    counts = [-(-k // case["page"]) for k in kv]
    n_pages = sum(counts) + 5
    k_pages, v_pages = cache_of(case, g, n_pages)
    return {"q": normal(g, (sum(new), case["heads"], case["dim"]), DTYPES[case["type"]]), "k_pages": k_pages, "v_pages": v_pages,
            "table": scattered(g, n_pages, counts, max(counts)), "cu": packed(new), "kv_len": ints(kv), "max_new": max(new), "max_kv": max(kv)}


def prepare_prefix(case, g):
    """What forking leaves: full pages of a prefix are shared, a partly filled last one is every sequence's own copy."""
    prefix, kv = prefix_lengths(case)
    page, per = case["page"], case["seqs"]
    n = case["groups"] * per
    full = [prefix[i // per] // page for i in range(n)]
    counts = [-(-kv[i] // page) - full[i] for i in range(n)]
    firsts = [prefix[j] // page for j in range(case["groups"])]
    n_pages = sum(counts) + sum(firsts) + 5
    k_pages, v_pages = cache_of(case, g, n_pages)
    width = max(f + c for f, c in zip(full, counts))
    pages = scattered(g, n_pages, firsts + counts, width)
    shared, tails = pages[: case["groups"]].repeat_interleave(per, 0), pages[case["groups"]:]
    at, held = torch.arange(width, device="cuda")[None, :], ints(full)[:, None]
    table = torch.where(at < held, shared, torch.gather(tails, 1, (at - held).clamp(0, width - 1).long()))
    table = torch.where(at < held + ints(counts)[:, None], table, -1).to(torch.int32).contiguous()
    # the copies of partly filled pages
    part = [(i - i % per, i) for i in range(n) if i % per and prefix[i // per] % page]
    if part:
        src, dst = (table.gather(1, ints(full)[:, None].long())[[p[k] for p in part], 0].long() for k in range(2))
        for pages in (k_pages, v_pages):
            raw = pages.view(torch.uint8)
            raw[dst] = raw[src]
    new = case["new"]
    return {"q": normal(g, (n * new, case["heads"], case["dim"]), DTYPES[case["type"]]), "k_pages": k_pages, "v_pages": v_pages, "table": table,
            "cu": packed([new] * n), "kv_len": ints(kv), "cu_group": packed([per] * case["groups"]), "prefix": ints(prefix),
            "max_prefix": max(prefix), "max_tail": max(kv[i] - prefix[i // per] for i in range(n))}


# ------------------------------------------------------------------ one pass


def run(s):
    if own:
        return {"append": own_append, "read": own_read, "attend": own_attend, "prefix": own_prefix}[s["case"]["op"]](s)
    return {"append": plain_append, "read": plain_read, "attend": plain_attend, "prefix": plain_prefix}[s["case"]["op"]](s)


def own_append(s):
    import heteromm_b200 as hmm
    c = s["case"]
    q, k, v = s["qkv"].split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)
    q = hmm.paged_quant_append(q, k, v, s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], s["rope"], q_weight=s["q_weight"],
                               k_weight=s["k_weight"], interleaved=c["interleaved"], out=s["out"], status=s["status"])
    k, v = hmm.paged_quant_read(s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], k.shape[0], dtype=DTYPES[c["type"]], status=s["status"])
    return q, k, v


def own_read(s):
    import heteromm_b200 as hmm
    return hmm.paged_quant_read(s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], s["rows"], dtype=DTYPES[s["case"]["type"]], status=s["status"])


def own_attend(s):
    import heteromm_b200 as hmm
    c = s["case"]
    return hmm.paged_quant_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], window=c["window"], sinks=c["sinks"],
                                     max_new=s["max_new"], return_lse=c["lse"], status=s["status"])


def own_prefix(s):
    import heteromm_b200 as hmm
    c = s["case"]
    return hmm.paged_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], s["cu_group"], s["prefix"],
                                      max_new=c["new"], return_lse=c["lse"], status=s["status"])


def owners(cu, total):
    """The sequence of each of the batch's tokens, and its number within it."""
    at = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), at.to(cu.dtype), right=True)
    return seq, at - cu.long()[seq]


def rows_of(pages, kind, table, seq, pos):
    """fp32 values [..., heads, D] of the tokens at `pos` of sequences `seq`."""
    t = pages.shape[2]
    phys, row = table.long()[seq, pos // t].clamp(min=0), pos % t
    if kind == "16":
        return pages[phys, :, row].float()
    codes, scales = parts(pages)
    return values(codes[phys, :, row], scales[phys, :, row], kind)


def rotated(x, angle, interleaved):
    """x with its first 2 * angle.shape[1] values turned in pairs; angle [tokens, pairs, (cos, sin)]."""
    half = angle.shape[1]
    cos, sin = angle[:, None, :, 0], angle[:, None, :, 1]
    part, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = part[..., :half], part[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def plain_append(s):
    c, kind = s["case"], s["case"]["cache"]
    q, k, v = s["qkv"].split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)
    seq, j = owners(s["cu"], q.shape[0])
    cu, kv_len = s["cu"].long(), s["kv_len"].long()
    pos = (kv_len - cu[1:] + cu[:-1])[seq] + j

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        return rotated(x, s["rope"][pos], c["interleaved"])

    def stored(x, pages):
        codes, scales = parts(pages)
        phys, row = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
        codes[phys, :, row], scales[phys, :, row] = quantised(x, kind)
        return rows_of(pages, kind, s["table"], seq, pos).to(q.dtype)

    s["out"].copy_(turned(q, s["q_weight"]))
    return s["out"], stored(turned(k, s["k_weight"]), s["k_pages"]), stored(v.float(), s["v_pages"])


def plain_read(s):
    c = s["case"]
    seq, pos = owners(s["cu"], s["rows"])
    return tuple(rows_of(s[p], c["cache"], s["table"], seq, pos).to(DTYPES[c["type"]]) for p in ("k_pages", "v_pages"))


def plain_attend(s):
    c, q, cu, kv_len = s["case"], s["q"], s["cu"].long(), s["kv_len"].long()
    n, hk, g, d = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    new, kv = s["max_new"], s["max_kv"]
    key = torch.arange(kv, device=q.device)
    inside = key[None, :] < kv_len[:, None]
    held = torch.where(inside, key, 0)
    every = torch.arange(n, device=q.device)[:, None]
    k = rows_of(s["k_pages"], c["cache"], s["table"], every, held).transpose(1, 2)
    v = rows_of(s["v_pages"], c["cache"], s["table"], every, held).transpose(1, 2)
    rows = (cu[:-1, None] + torch.arange(new, device=q.device)).clamp(max=q.shape[0] - 1)
    qp = q[rows].float().reshape(n, new, hk, g, d).permute(0, 2, 1, 3, 4).reshape(n, hk, new * g, d)
    score = (qp @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).reshape(n, hk, new, g, kv)
    pos = (kv_len - (cu[1:] - cu[:-1]))[:, None] + torch.arange(new, device=q.device)
    seen = (key <= pos[..., None]) & inside[:, None, :]
    if c["window"]:
        seen &= (key > pos[..., None] - c["window"]) | (key < c["sinks"])
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(n, hk, new * g, kv) @ v).reshape(n, hk, new, g, d) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1)
    seq, j = owners(s["cu"], q.shape[0])
    out = o[seq, :, j].reshape(q.shape).to(q.dtype)
    return (out, lse[seq, :, j].reshape(q.shape[:2])) if c["lse"] else out


def plain_prefix(s):
    """Scores of a group's rows over its prefix and of each sequence's over its own tail, under one softmax."""
    c, q, kind = s["case"], s["q"], s["case"]["cache"]
    groups, per, new, hk, g, d = c["groups"], c["seqs"], c["new"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    n, prefix = groups * per, s["prefix"].long()
    at = torch.arange(s["max_prefix"], device=q.device)
    first = s["cu_group"].long()[:-1, None]
    near = at < prefix[:, None]
    k1, v1 = (rows_of(s[p], kind, s["table"], first, torch.where(near, at, 0)).transpose(1, 2) for p in ("k_pages", "v_pages"))
    own_prefix_len = prefix.repeat_interleave(per)[:, None]
    behind = own_prefix_len + torch.arange(s["max_tail"], device=q.device)
    far = behind < s["kv_len"].long()[:, None]
    every = torch.arange(n, device=q.device)[:, None]
    k2, v2 = (rows_of(s[p], kind, s["table"], every, torch.where(far, behind, 0)).transpose(1, 2) for p in ("k_pages", "v_pages"))
    qs = q.float().reshape(n, new, hk, g, d).permute(0, 2, 1, 3, 4)
    qg = qs.reshape(groups, per, hk, new * g, d).transpose(1, 2).reshape(groups, hk, per * new * g, d)
    x1 = (qg @ k1.transpose(-1, -2)).masked_fill_(~near[:, None, None, :], -math.inf)
    x2 = (qs.reshape(n, hk, new * g, d) @ k2.transpose(-1, -2)).reshape(n, hk, new, g, -1)
    pos = s["kv_len"].long()[:, None] - new + torch.arange(new, device=q.device)
    x2.masked_fill_(~(far[:, None, :] & (behind[:, None, :] <= pos[..., None]))[:, None, :, None, :], -math.inf)

    def by_sequence(x):   # [groups, hk, per * new * g, ...] -> [n, hk, new * g, ...]
        return x.reshape(groups, hk, per, new * g, -1).transpose(1, 2).reshape(n, hk, new * g, -1)

    def by_group(x):
        return x.reshape(groups, per, hk, new * g, -1).transpose(1, 2).reshape(groups, hk, per * new * g, -1)

    scale = 1.0 / math.sqrt(d)
    x2 = x2.reshape(n, hk, new * g, -1).mul_(scale)
    x1.mul_(scale)
    top = torch.maximum(by_sequence(x1.amax(-1)), x2.amax(-1, keepdim=True))
    p1, p2 = x1.sub_(by_group(top)).exp_(), x2.sub_(top).exp_()
    total = by_sequence(p1.sum(-1)) + p2.sum(-1, keepdim=True)
    o = (by_sequence(p1 @ v1) + p2 @ v2) / total
    out = o.reshape(n, hk, new, g, d).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)
    lse = (top + total.log()).reshape(n, hk, new, g).transpose(1, 2).reshape(q.shape[:2])
    return (out, lse) if c["lse"] else out


# ------------------------------------------------------------------ what a pass cannot do without


def row_bytes(case):
    """A token's key and value of one head."""
    d = case["dim"]
    return 4 * d if case["cache"] == "16" else 2 * (d + d // GROUP)


def work(case):
    d = case["dim"]
    if case["op"] == "append":  # q, k and v read, q and the cache written, the stored rows read and given back
        new, _ = lengths(dict(case, ragged=False))
        tokens = sum(new)
        values_ = tokens * (case["heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": 4 * values_ + 2 * tokens * case["kv_heads"] * row_bytes(case) + 4 * case["rotary"] * tokens, "flops": 8 * values_}
    if case["op"] == "read":
        tokens = sum(read_lengths(case))
        return {"bytes": tokens * case["kv_heads"] * (row_bytes(case) + 4 * d), "flops": 2 * tokens * case["kv_heads"] * d}
    if case["op"] == "prefix":
        prefix, kv = prefix_lengths(case)
        new, per = case["new"], case["seqs"]
        tails = [k - prefix[i // per] for i, k in enumerate(kv)]
        pairs = sum(new * prefix[i // per] + new * t - new * (new - 1) // 2 for i, t in enumerate(tails))
        tokens = len(kv) * new
        return {"bytes": (sum(prefix) + sum(tails)) * case["kv_heads"] * row_bytes(case) + 4 * tokens * case["heads"] * d + (4 * tokens * case["heads"] if case["lse"] else 0),
                "flops": 4 * d * case["heads"] * pairs}
    new, kv = lengths(case)
    tokens = sum(new)
    pairs, read = 0, 0
    for n, k in zip(new, kv):
        first = k - n + 1  # keys that the first new token sees
        w = case["window"] + case["sinks"] if case["window"] else k
        flat = max(0, min(n, k - max(first, w) + 1)) if k > w else 0  # tokens that see as many keys as window and first tokens have
        rising = n - flat
        pairs += flat * w + rising * first + rising * (rising - 1) // 2
        read += min(k, w + n) if case["window"] else k
    return {"bytes": 4 * d * tokens * case["heads"] + read * case["kv_heads"] * row_bytes(case) + (4 * tokens * case["heads"] if case["lse"] else 0),
            "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": exact_append, "read": exact_read, "attend": exact_attend, "prefix": exact_prefix}[case["op"]](case, s)


E4M3 = [(1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) if b >> 3 else (b & 7) / 8 * 2.0 ** -6 for b in range(127)]  # codes 0 ... 126; 127 is NaN


def exact_rows(case, pages, table, i, positions):
    """Values in 64 bits of tokens of sequence i, [tokens, heads, D], looked up code by code."""
    t = case["page"]
    phys, row = table[i].long()[positions // t], positions % t
    if case["cache"] == "16":
        return pages[phys, :, row].double()
    n, h, _, width = pages.shape
    d = case["dim"]
    raw = pages.view(torch.uint8).reshape(n, h, t * width)[phys]
    byte = torch.gather(raw, 2, (row[:, None, None] * d + torch.arange(d, device="cuda")).expand(-1, h, -1)).long()
    scale = torch.gather(raw, 2, (t * d + row[:, None, None] * (d // GROUP) + torch.arange(d, device="cuda") // GROUP).expand(-1, h, -1)).double()
    if case["cache"] == "int8":
        value = (byte - 256 * (byte >= 128)).double()
    else:
        grid = torch.tensor(E4M3 + [math.nan], dtype=torch.float64, device="cuda")
        value = grid[byte & 127] * torch.where(byte >= 128, -1.0, 1.0).double()
    return value * torch.pow(2.0, scale - 127)


def exact_quantised(x, kind):
    """x in 64 bits [tokens, heads, D] as the nearest values on the grid of each 32's scale, ties to the even code."""
    y = x.reshape(*x.shape[:2], -1, GROUP)
    top = y.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** HIGHEST)
    for e in range(HIGHEST, LOWEST[kind] - 1, -1):
        scale = torch.where(top <= LARGEST[kind] * 2.0 ** e, 2.0 ** e, scale)
    z = (y / scale).clamp(-LARGEST[kind], LARGEST[kind])
    if kind == "e4m3":  # steps of an eighth of the value's power of two, at least 2^-9
        step = torch.pow(2.0, torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6)))) / 8
        z = torch.round(z / step) * step
    else:
        z = torch.round(z)
    return (z * scale).reshape(x.shape)


def exact_append(case, s):
    new, kv = lengths(dict(case, ragged=False))
    hq, hk, half = case["heads"], case["kv_heads"], case["rotary"] // 2
    x = s["qkv"].double()
    y = x[:, : hq + hk]
    if case["norm"]:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6)
        y = torch.cat([y[:, :hq] * s["q_weight"].double(), y[:, hq:] * s["k_weight"].double()], 1)
    pos = torch.cat([torch.arange(k - n, k, device="cuda") for n, k in zip(new, kv)])
    # pairs as complex numbers, turned by the table's angle
    turn = torch.view_as_complex(s["rope"].double())[pos][:, None, :]
    part = y[..., : 2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
    part = part if case["interleaved"] else part.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    z = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    y = torch.cat([z, y[..., 2 * half:]], -1)
    return y[:, :hq], exact_quantised(y[:, hq:], case["cache"]), exact_quantised(x[:, hq + hk:], case["cache"])


def exact_read(case, s):
    kv = read_lengths(case)
    return tuple(torch.cat([exact_rows(case, s[p], s["table"], i, torch.arange(k, device="cuda")) for i, k in enumerate(kv)]) for p in ("k_pages", "v_pages"))


def exact_sequence(case, s, i, start, n, length, window, sinks, out, lse):
    hk, g, d = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    keys, vals = (exact_rows(case, s[p], s["table"], i, torch.arange(length, device="cuda")) for p in ("k_pages", "v_pages"))
    for h in range(hk):
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            q = s["q"][start + a: start + b, h * g: (h + 1) * g].double()
            x = torch.einsum("tgd,kd->tgk", q, keys[:, h]) / math.sqrt(d)
            p = torch.arange(length - n + a, length - n + b, device="cuda")[:, None, None]
            k = torch.arange(length, device="cuda")[None, None, :]
            hide = k > p
            if window:
                hide = hide | ((k <= p - window) & (k >= sinks))
            x = torch.where(hide, -math.inf, x)
            out[start + a: start + b, h * g: (h + 1) * g] = torch.softmax(x, -1) @ vals[:, h]
            lse[start + a: start + b, h * g: (h + 1) * g] = torch.logsumexp(x, -1)


def exact_attend(case, s):
    new, kv = lengths(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    start = 0
    for i, (n, length) in enumerate(zip(new, kv)):
        exact_sequence(case, s, i, start, n, length, case["window"], case["sinks"], out, lse)
        start += n
    return (out, lse) if case["lse"] else out


def exact_prefix(case, s):
    """Each sequence by itself, over all of its own tokens."""
    _, kv = prefix_lengths(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for i, length in enumerate(kv):
        exact_sequence(case, s, i, i * case["new"], case["new"], length, 0, 0, out, lse)
    return (out, lse) if case["lse"] else out

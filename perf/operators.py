"""The operators of a served paged KV cache with several heads, as measured cases.

Three operators work on one cache, K and V page arrays [n_pages, n_kv_heads, page_tokens, D]:

  attention  a chunk of new tokens of each sequence attends over its paged cache (one token for
             decoding, a few drafted ones, a whole prompt), causal, with an optional sliding
             window beside a few first tokens that stay visible
  append     RMS norm of each query and key head, position rotation, and the store of keys and
             values into the cache's pages, in one pass
  turn,      the cache's housekeeping: copying pages, forking, growing and freeing sequences
  compact    (turn), and moving the live pages to the front of the cache (compact)

`run` computes them in elementary torch operations, or (own) by the calls a user makes.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one conversation decoding one token: all latency
        {"name": "attention one token", "op": "attention", "type": "bf16", "seqs": 1, "new": 1, "kv": 777, "ragged": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": False},
        # a decoding batch of ragged long contexts: bound by reading the cache
        {"name": "attention decode batch", "op": "attention", "type": "bf16", "seqs": 64, "new": 1, "kv": 16384, "ragged": True, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": False},
        # verifying drafted tokens, seven query heads to a key head
        {"name": "attention drafted", "op": "attention", "type": "fp16", "seqs": 16, "new": 5, "kv": 5001, "ragged": True, "heads": 28, "kv_heads": 4,
         "dim": 128, "page": 32, "window": 0, "sinks": 0, "lse": True},
        # a step that mixes the chunk of one prompt with decoding sequences
        {"name": "attention mixed step", "op": "attention", "type": "bf16", "seqs": 8, "new": 1001, "kv": 4096, "ragged": True, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": False},
        # a whole long prompt: bound by the matrix products
        {"name": "attention prompt", "op": "attention", "type": "bf16", "seqs": 1, "new": 8192, "kv": 8192, "ragged": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "sinks": 0, "lse": True},
        # chunks of streaming sequences: a window beside the first tokens
        {"name": "attention window", "op": "attention", "type": "fp16", "seqs": 4, "new": 2000, "kv": 16000, "ragged": True, "heads": 16, "kv_heads": 16,
         "dim": 64, "page": 64, "window": 1024, "sinks": 4, "lse": False},
        # the step before the attention of a decoding batch: half of each head turned, in neighbouring pairs
        {"name": "append decode batch", "op": "append", "type": "fp16", "seqs": 64, "new": 1, "kv": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "rotary": 64, "interleaved": True, "norm": True},
        # the chunks of two prompts
        {"name": "append prompt", "op": "append", "type": "bf16", "seqs": 2, "new": 4099, "kv": 5000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "rotary": 128, "interleaved": False, "norm": True},
        # a small server between two steps
        {"name": "turn small", "op": "turn", "type": "bf16", "seqs": 8, "pages": 512, "kv": 300, "kv_heads": 2, "dim": 64, "page": 16, "copied": 16},
        # a large one
        {"name": "turn large", "op": "turn", "type": "bf16", "seqs": 256, "pages": 20000, "kv": 1500, "kv_heads": 8, "dim": 128, "page": 16, "copied": 1024},
        # a fragmented cache put together again
        {"name": "compact small", "op": "compact", "type": "bf16", "seqs": 8, "pages": 300, "live": 0.4, "kv_heads": 2, "dim": 64, "page": 16},
        {"name": "compact large", "op": "compact", "type": "bf16", "seqs": 256, "pages": 30000, "live": 0.5, "kv_heads": 8, "dim": 128, "page": 16},
    ]


def spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "append", "turn", "compact"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "attention":
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        c = {"op": op, "type": dtype, "seqs": spread(rng, 1, 64), "new": spread(rng, 1, 4096), "kv": 0, "ragged": rng.random() < 0.7,
             "heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([64, 64, 80, 128, 128, 128, 256]), "page": rng.choice([8, 16, 16, 24, 32, 64, 128]),
             "window": 0, "sinks": 0, "lse": rng.random() < 0.5}
        c["kv"] = c["new"] + spread(rng, 1, 16384) - 1
        if rng.random() < 0.4:
            c["window"], c["sinks"] = spread(rng, 16, 4096), rng.choice([0, 1, 4, 33])
        while c["seqs"] * c["new"] * c["heads"] * c["kv"] > 1 << 30 or c["seqs"] * c["kv_heads"] * c["kv"] * c["dim"] > 1 << 30:
            if c["seqs"] > 1:
                c["seqs"] = c["seqs"] // 2
            else:
                c["new"], c["kv"] = (c["new"] + 1) // 2, c["kv"] // 2 + 1
        return c
    if op == "append":
        kv_heads, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 80, 128, 128, 256])
        c = {"op": op, "type": dtype, "seqs": spread(rng, 1, 128), "new": spread(rng, 1, 4096), "kv": 0, "heads": kv_heads * rng.choice([1, 2, 4, 7]),
             "kv_heads": kv_heads, "dim": dim, "page": rng.choice([8, 16, 16, 24, 64]), "rotary": rng.choice([dim, dim, dim // 2, 20]),
             "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.7}
        while c["seqs"] * c["new"] > 8192:
            c["seqs"], c["new"] = (c["seqs"] + 1) // 2, (c["new"] + 1) // 2
        c["kv"] = c["new"] + spread(rng, 1, 2048) - 1
        return c
    heads, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128]), rng.choice([8, 16, 16, 24, 64])
    if op == "turn":
        seqs, kv, copied = spread(rng, 4, 256), spread(rng, 20, 2000), spread(rng, 1, 512)
        while seqs > 4 and 2 * seqs * (kv // page + 3) * page * heads * dim > 1 << 29:
            seqs //= 2
        return {"op": op, "type": dtype, "seqs": seqs, "pages": 2 * seqs * (kv // page + 3) + 3 * copied + 8, "kv": kv, "kv_heads": heads, "dim": dim, "page": page,
                "copied": copied}
    pages = min(spread(rng, 256, 30000), (1 << 29) // (page * heads * dim))
    return {"op": op, "type": dtype, "seqs": spread(rng, 1, 256), "pages": pages, "live": round(rng.uniform(0.1, 0.9), 3), "kv_heads": heads, "dim": dim, "page": page}


def lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence: a part of the case, not of the seed."""
    r = random.Random(case["seqs"] * 7919 + case["kv"])
    new, kv = [], []
    for i in range(case["seqs"]):
        n = case["new"]
        if case.get("ragged", True) and n > 8 and i > 0:
            n = 1 if i % 2 else max(1, int(n * r.uniform(0.0, 0.25)))  # a chunk beside decoding sequences and short prompts
        k = case["kv"] if i == 0 or not case.get("ragged", True) else int(case["kv"] * r.uniform(0.05, 1.0))
        new.append(n)
        kv.append(max(n, k))
    return new, kv


# ------------------------------------------------------------------ inputs


def normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cache_of(case, g, n_pages):
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    return normal(g, shape, DTYPES[case["type"]]), normal(g, shape, DTYPES[case["type"]])


def scattered(g, n_pages, counts, width):
    """A page table whose rows hold `counts` pages each, taken from shuffled pages; -1 behind them."""
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([0] + counts[:-1], device="cuda").cumsum(0)
    at = torch.arange(width, device="cuda")[None, :]
    held = at < torch.tensor(counts, device="cuda")[:, None]
    table = torch.where(held, perm[(first[:, None] + at).clamp(max=n_pages - 1)], -1)
    return table.to(torch.int32), perm


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"attention": prepare_attention, "append": prepare_append, "turn": prepare_turn, "compact": prepare_compact}[case["op"]](case, g)


def prepare_attention(case, g):
    new, kv = lengths(case)
    page, dtype = case["page"], DTYPES[case["type"]]
    counts = [-(-k // page) for k in kv]
    n_pages = sum(counts) + 5
    k_pages, v_pages = cache_of(case, g, n_pages)
    table, _ = scattered(g, n_pages, counts, max(counts))
    total = sum(new)
    return {"case": case, "q": normal(g, (total, case["heads"], case["dim"]), dtype), "k_pages": k_pages, "v_pages": v_pages, "table": table,
            "cu": ints([0] + new).cumsum(0).to(torch.int32), "kv_len": ints(kv), "max_new": max(new), "max_kv": max(kv),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def prepare_append(case, g):
    new, kv = lengths(dict(case, ragged=False))
    page, dtype, half = case["page"], DTYPES[case["type"]], case["rotary"] // 2
    counts = [-(-k // page) for k in kv]
    # a decoding batch writes its last pages alone: only they are in the cache here, the table's earlier entries point at them too
    tail = [min(c, -(-n // page) + 1) for c, n in zip(counts, new)]
    n_pages = sum(tail) + 3
    k_pages, v_pages = cache_of(case, g, n_pages)
    last, _ = scattered(g, n_pages, tail, max(tail))
    width = max(counts)
    at = torch.arange(width, device="cuda")[None, :] - (ints(counts) - ints(tail))[:, None]
    table = torch.gather(last, 1, at.clamp(0, max(tail) - 1).long()).to(torch.int32).contiguous()
    total, hq, hk, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    qkv = normal(g, (total, hq + 2 * hk, d), dtype, 2.0)  # the output of one projection
    turn = torch.arange(max(kv), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)[None, :]
    return {"case": case, "qkv": qkv, "k_pages": k_pages, "v_pages": v_pages, "table": table, "cu": ints([0] + new).cumsum(0).to(torch.int32),
            "kv_len": ints(kv), "rope": torch.stack([turn.cos(), turn.sin()], -1).float().contiguous(),
            "q_weight": (1 + 0.1 * normal(g, (d,), torch.float32)).to(dtype) if case["norm"] else None,
            "k_weight": (1 + 0.1 * normal(g, (d,), torch.float32)).to(dtype) if case["norm"] else None,
            "out": torch.empty((total, hq, d), dtype=dtype, device="cuda"), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def prepare_turn(case, g):
    """A server's state: `seqs` rows, of which a quarter are empty and an eighth finished; some prefixes saved in pages of their own."""
    seqs, page, n_pages, copied = case["seqs"], case["page"], case["pages"], case["copied"]
    r = random.Random(seqs * 31 + case["kv"])
    empty = max(1, seqs // 4)
    kv = [0 if s >= seqs - empty else max(1, int(case["kv"] * r.uniform(0.3, 1.0))) for s in range(seqs)]
    counts = [-(-k // page) for k in kv]
    k_pages, v_pages = cache_of(case, g, n_pages)
    width = max(counts) + 8
    table, perm = scattered(g, n_pages, counts, width)
    used = sum(counts)
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[perm[: used + 2 * copied].long()] = 1  # the rows' pages, the saved ones and where they go
    done = list(range(0, seqs - empty, 8))
    live = [s for s in range(seqs - empty) if s % 8]
    fork_dst = list(range(seqs - empty, seqs))
    fork_src = [live[(3 * i) % len(live)] for i in range(empty)]
    grown = [0 if s in done else 1 + (s * 5) % (2 * page) for s in range(seqs)]
    return {"case": case, "k_pages": k_pages, "v_pages": v_pages, "table": table, "refs": refs, "kv_len": ints(kv), "src": perm[used: used + copied].contiguous(),
            "dst": perm[used + copied: used + 2 * copied].contiguous(), "done": ints(done), "fork_src": ints(fork_src), "fork_dst": ints(fork_dst),
            "grown": ints(grown), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def prepare_compact(case, g):
    n_pages, seqs = case["pages"], case["seqs"]
    live = live_pages(case)
    per = [live // seqs + (1 if s < live % seqs else 0) for s in range(seqs)]
    k_pages, v_pages = cache_of(case, g, n_pages)
    table, perm = scattered(g, n_pages, per, max(per) + 2)
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[perm[:live].long()] = 1
    if seqs > 1 and per[0] > 0 and per[1] > 0:  # the second row shares the first one's first page
        refs[table[1, 0].long()] = 0
        table[1, 0] = table[0, 0]
        refs[table[0, 0].long()] = 2
    return {"case": case, "k_pages": k_pages, "v_pages": v_pages, "table": table, "refs": refs, "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def live_pages(case):
    return max(1, int(case["pages"] * case["live"]))


# ------------------------------------------------------------------ one pass


def run(s):
    if own:
        return {"attention": own_attention, "append": own_append, "turn": own_turn, "compact": own_compact}[s["case"]["op"]](s)
    return {"attention": plain_attention, "append": plain_append, "turn": plain_turn, "compact": plain_compact}[s["case"]["op"]](s)


def own_attention(s):
    import heteromm_b200 as hmm
    c = s["case"]
    return hmm.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], window=c["window"], sinks=c["sinks"],
                               max_new=s["max_new"], return_lse=c["lse"], status=s["status"])


def own_append(s):
    import heteromm_b200 as hmm
    c = s["case"]
    q, k, v = s["qkv"].split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)
    q = hmm.paged_kv_append(q, k, v, s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], s["rope"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                            interleaved=c["interleaved"], out=s["out"], status=s["status"])
    return q, s["k_pages"], s["v_pages"]


def own_turn(s):
    import heteromm_b200 as hmm
    hmm.paged_copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"], status=s["status"])
    table, refs, kv_len = hmm.paged_free(s["table"], s["refs"], s["kv_len"], s["done"], status=s["status"])
    table, refs, kv_len = hmm.paged_fork(table, refs, kv_len, s["fork_src"], s["fork_dst"], s["k_pages"], s["v_pages"], status=s["status"])
    table, refs, kv_len = hmm.paged_grow(table, refs, kv_len, s["grown"], s["case"]["page"], status=s["status"])
    return table, refs, kv_len, s["k_pages"], s["v_pages"]


def own_compact(s):
    import heteromm_b200 as hmm
    table, refs, live = hmm.paged_compact(s["table"], s["refs"], s["k_pages"], s["v_pages"], status=s["status"])
    return table, refs, live, s["k_pages"], s["v_pages"]


def owners(cu, total):
    """The sequence of each of the batch's tokens, and its number within it."""
    at = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), at.to(cu.dtype), right=True)
    return seq, at - cu.long()[seq]


def plain_attention(s):
    c, q, table, cu, kv_len = s["case"], s["q"], s["table"], s["cu"].long(), s["kv_len"].long()
    n, hk, g, d, page = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["page"]
    new, kv = s["max_new"], s["max_kv"]
    held = table.long().clamp(min=0)

    def gathered(pages):
        return pages[held].permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)[:, :, :kv].float()

    key = torch.arange(kv, device=q.device)
    inside = key[None, :] < kv_len[:, None]
    k = gathered(s["k_pages"])
    v = gathered(s["v_pages"]) * inside[:, None, :, None]
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
    c = s["case"]
    q, k, v = s["qkv"].split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)
    seq, j = owners(s["cu"], q.shape[0])
    cu, kv_len = s["cu"].long(), s["kv_len"].long()
    pos = (kv_len - cu[1:] + cu[:-1])[seq] + j

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        return rotated(x, s["rope"][pos], c["interleaved"])

    phys, row = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    s["k_pages"][phys, :, row] = turned(k, s["k_weight"]).to(k.dtype)
    s["v_pages"][phys, :, row] = v
    s["out"].copy_(turned(q, s["q_weight"]))
    return s["out"], s["k_pages"], s["v_pages"]


def plain_turn(s):
    c, page = s["case"], s["case"]["page"]
    k_pages, v_pages = s["k_pages"], s["v_pages"]
    table, refs, kv_len = s["table"].clone(), s["refs"].clone(), s["kv_len"].clone()
    # copy
    k_pages[s["dst"].long()] = k_pages[s["src"].long()]
    v_pages[s["dst"].long()] = v_pages[s["src"].long()]
    # free: one reference less for each page that a finished row holds
    done = s["done"].long()
    count(refs, table[done], -1)
    table[done] = -1
    kv_len[done] = 0
    # fork: full pages are shared, the last one is copied where it is not full
    src, dst = s["fork_src"].long(), s["fork_dst"].long()
    length = kv_len[src].long()
    at = torch.arange(table.shape[1], device=table.device)
    shared = torch.where(at < (length // page)[:, None], table[src], -1)
    partial = length % page != 0
    rank = torch.where(partial, partial.cumsum(0) - 1, partial.sum() + (~partial).cumsum(0) - 1)
    got = free_pages(refs)[rank].to(torch.int32)  # those without a partial page copy a free page onto itself
    old = table[src, (length // page).clamp(max=table.shape[1] - 1)]
    old, got = torch.where(partial, old, got), got
    k_pages[got.long()] = k_pages[old.long()]
    v_pages[got.long()] = v_pages[old.long()]
    table[dst] = torch.where((at == (length // page)[:, None]) & partial[:, None], got[:, None], shared)
    count(refs, table[dst], 1)
    kv_len[dst] = kv_len[src]
    # grow: the entries that the new tokens need and no page holds yet
    to = kv_len + s["grown"]
    missing = (at < ((to + page - 1) // page)[:, None]) & (at >= (kv_len // page)[:, None]) & (table < 0)
    order = (missing.flatten().cumsum(0) - 1).clamp(min=0).reshape(table.shape)
    taken = free_pages(refs)[order.clamp(max=refs.shape[0] - 1)].to(torch.int32)
    table = torch.where(missing, taken, table)
    count(refs, torch.where(missing, taken, -1), 1)
    return table, refs, to, k_pages, v_pages


def count(refs, pages, by):
    """Adds `by` to the references of every page in `pages` (entries below 0 are none)."""
    pages = pages.flatten().long()
    refs.scatter_add_(0, pages.clamp(min=0), torch.where(pages >= 0, by, 0).to(refs.dtype))


def free_pages(refs):
    """All pages, those without references first, in ascending order."""
    return torch.sort((refs != 0).to(torch.int8), stable=True).indices


def plain_compact(s):
    table, refs, k_pages, v_pages = s["table"], s["refs"], s["k_pages"], s["v_pages"]
    n = refs.shape[0]
    page = torch.arange(n, device=refs.device)
    used = refs != 0
    live = used.sum()
    front = page < live
    # the k-th live page behind the front goes to the k-th free one in it
    src = torch.nonzero(used & ~front).flatten()
    dst = torch.nonzero(~used & front).flatten()
    k_pages[dst] = k_pages[src]
    v_pages[dst] = v_pages[src]
    to = page.clone()
    to[src] = dst
    new_refs = torch.where(front, refs, 0)
    new_refs[dst] = refs[src]
    new_table = torch.where(table >= 0, to[table.long().clamp(min=0)].to(torch.int32), table)
    return new_table, new_refs, live.to(torch.int32).reshape(1), k_pages, v_pages


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    size, d = 2, case["dim"]
    if case["op"] == "attention":
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
        return {"bytes": size * d * (2 * tokens * case["heads"] + 2 * read * case["kv_heads"]) + (4 * tokens * case["heads"] if case["lse"] else 0),
                "flops": 4 * d * case["heads"] * pairs}
    if case["op"] == "append":
        new, _ = lengths(dict(case, ragged=False))
        values = sum(new) * (case["heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": 2 * size * values + 4 * case["rotary"] * sum(new), "flops": 8 * values}
    page_bytes = 2 * size * case["kv_heads"] * case["page"] * d
    if case["op"] == "turn":
        forks = max(1, case["seqs"] // 4)
        table = 4 * case["seqs"] * (case["kv"] // case["page"] + 9)
        return {"bytes": 2 * page_bytes * (case["copied"] + forks) + 2 * 4 * case["pages"] + 2 * table, "flops": 0}
    live = live_pages(case)
    moved = live * (case["pages"] - live) / case["pages"]
    return {"bytes": 2 * page_bytes * moved + 2 * 4 * case["pages"] + 2 * 4 * live, "flops": 0}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    if case["op"] == "attention":
        return exact_attention(case, prepare(case, seed))
    if case["op"] == "append":
        return exact_append(case, prepare(case, seed))
    return None  # whole numbers, and pages that are moved as they are


def exact_attention(case, s):
    new, kv = lengths(case)
    hk, g, d, page = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    start = 0
    for i, (n, length) in enumerate(zip(new, kv)):
        ids = s["table"][i, : -(-length // page)].long()
        for h in range(hk):
            keys = s["k_pages"][ids, h].reshape(-1, d)[:length].double()
            values = s["v_pages"][ids, h].reshape(-1, d)[:length].double()
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                q = s["q"][start + a: start + b, h * g: (h + 1) * g].double()
                x = torch.einsum("tgd,kd->tgk", q, keys) / math.sqrt(d)
                p = torch.arange(length - n + a, length - n + b, device="cuda")[:, None, None]
                k = torch.arange(length, device="cuda")[None, None, :]
                hide = k > p
                if case["window"]:
                    hide = hide | ((k <= p - case["window"]) & (k >= case["sinks"]))
                x = torch.where(hide, -math.inf, x)
                out[start + a: start + b, h * g: (h + 1) * g] = torch.softmax(x, -1) @ values
                lse[start + a: start + b, h * g: (h + 1) * g] = torch.logsumexp(x, -1)
        start += n
    return (out, lse) if case["lse"] else out


def exact_append(case, s):
    new, kv = lengths(dict(case, ragged=False))
    hq, hk, half, page = case["heads"], case["kv_heads"], case["rotary"] // 2, case["page"]
    x = s["qkv"].double()
    if case["norm"]:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        y = torch.cat([y[:, :hq] * s["q_weight"].double(), y[:, hq: hq + hk] * s["k_weight"].double()], 1)
    else:
        y = x[:, : hq + hk]
    pos = torch.cat([torch.arange(k - n, k, device="cuda") for n, k in zip(new, kv)])
    # pairs as complex numbers, turned by the table's angle
    turn = torch.view_as_complex(s["rope"].double())[pos][:, None, :]
    part = y[..., : 2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
    part = part if case["interleaved"] else part.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    z = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    y = torch.cat([z, y[..., 2 * half:]], -1)
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(new)])
    phys, row = s["table"][seq, pos // page].long(), pos % page
    k_pages[phys, :, row] = y[:, hq:]
    v_pages[phys, :, row] = x[:, hq + hk:]
    return y[:, :hq], k_pages, v_pages

"""Sizes of the calls over a cache in 8 bits and over shared prefixes that lie at the ends: thousands of
sequences and groups, small and odd heads, pages longer than a tile of keys."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from test_prefix_attention_gpu import shared, with_join
from test_quant_attention_gpu import filled, run_case
from test_serve_attention_gpu import check, reference

pytestmark = pytest.mark.gpu


def spread_reference(q, k, v, table, new, kv, pick):
    """The reference of some sequences, and their rows."""
    first = np.concatenate([[0], np.cumsum(new)])
    rows = torch.cat([torch.arange(first[s], first[s + 1]) for s in pick]).to(q.device)
    return rows, with_join(reference(q[rows], k, v, table[pick], [new[s] for s in pick], [kv[s] for s in pick]))


@pytest.mark.parametrize("kind", [None, "e4m3"])
def test_thousands_of_sequences(cuda, kind):
    """3,000 sequences in 1,300 groups, of one to many; rows of every 37th are looked at."""
    rng = np.random.RandomState(3)
    n = 3000
    cuts = np.sort(np.concatenate([[0, 500], rng.choice(np.arange(501, n), 1298, replace=False), [n]]))    # one group of 500
    groups = [(int(a), int(b), int(rng.randint(0, 70))) for a, b in zip(cuts[:-1], cuts[1:])]
    new = rng.randint(0, 3, n).tolist()
    kv = [0] * n
    for a, b, p in groups:
        for s in range(a, b):
            kv[s] = p + new[s] + int(rng.randint(0, 20))
    hq, hk, d, pt = 4, 2, 64, 16
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 120, groups, new, kv, hq, hk, d, pt, torch.bfloat16, pad=4)
    kp, vp = k, v
    if kind:
        kp, vp, k, v = filled(k, v, kind)
    out, lse = hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, return_lse=True)
    rows, ref = spread_reference(q, k, v, table, new, kv, list(range(0, n, 37)))
    check(out[rows], lse[rows], ref)


def test_more_parts_than_sequences_may_be(cuda):
    """65,535 sequences, a group for each two: 98,302 parts."""
    n, pt, d = 65535, 16, 16
    new, kv = [1] * n, [20] * n
    g = torch.Generator(device=cuda).manual_seed(121)
    k, v = (torch.randn((2048, 1, pt, d), generator=g, device=cuda).to(torch.float16) for _ in range(2))
    q = torch.randn((n, 1, d), generator=g, device=cuda).to(torch.float16)
    table = torch.randint(0, 2048, (n, 2), generator=g, device=cuda, dtype=torch.int32)
    table[1:n - 1:2, 0] = table[0:n - 2:2, 0]
    cu, kv_len = torch.arange(n + 1, dtype=torch.int32, device=cuda), torch.full((n,), 20, dtype=torch.int32, device=cuda)
    cg = torch.arange(0, n, 2, dtype=torch.int32, device=cuda)
    pl = torch.full((cg.numel() - 1,), 16, dtype=torch.int32, device=cuda)
    out, lse = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, return_lse=True)
    rows, ref = spread_reference(q, k, v, table, new, kv, list(range(0, n, 1021)) + [n - 3, n - 2, n - 1])
    check(out[rows], lse[rows], ref)


@pytest.mark.parametrize("d", [8, 24, 72, 136, 248])
def test_odd_heads(cuda, d):
    groups, new, kv = [(0, 6, 130), (6, 9, 60)], [1, 2, 40, 1, 3, 1, 9, 1, 1], [140, 150, 300, 131, 135, 160, 90, 61, 75]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 122 + d, groups, new, kv, 6, 2, d, 16, torch.float16, pad=2)
    out, lse = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, return_lse=True)
    check(out, lse, with_join(reference(q, k, v, table, new, kv)))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", [  # new, kv, hq, hk, d, pt
    ([1, 1, 3], [900, 256, 700], 8, 2, 128, 256), ([100, 1, 40], [900, 256, 700], 8, 2, 128, 256),
    ([70, 1], [2300, 1999], 4, 2, 64, 1000), ([1, 2], [2300, 1999], 4, 2, 64, 1000),
    ([70, 1], [5000, 4097], 4, 1, 256, 4096), ([60, 5], [600, 433], 4, 2, 224, 144), ([1], [1], 64, 64, 32, 512),
])
def test_long_pages(cuda, shape, kind):
    run_case(cuda, 130, *shape, "bf16", kind, pad=3)
    run_case(cuda, 131, *shape, "fp16", kind, window=90, sinks=7)


@pytest.mark.parametrize("kind", [None, "int8"])
def test_a_prefix_of_long_pages(cuda, kind):
    groups, new, kv = [(0, 5, 777), (6, 9, 600)], [1, 2, 40, 1, 3, 5, 9, 1, 1], [800, 900, 1000, 778, 1300, 30, 609, 700, 1200]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 132, groups, new, kv, 8, 2, 128, 256, torch.bfloat16)
    kp, vp = k, v
    if kind:
        kp, vp, k, v = filled(k, v, kind)
    out, lse = hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, return_lse=True)
    check(out, lse, with_join(reference(q, k, v, table, new, kv)))

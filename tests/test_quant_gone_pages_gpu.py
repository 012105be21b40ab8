"""A page-table entry out of its bounds: the call is flagged, and the rows of the sequence that
names it are those over a page of zeros there, from both kernels and for both caches - nothing
of them comes from what a CTA's shared memory held before."""
import pytest
import torch

import heteromm_b200 as hmm
from test_prefix_attention_gpu import groups_of, with_join
from test_quant_attention_gpu import filled, long_table, raw
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu

KINDS = ["16", "e4m3", "int8"]


def hold(k, v, kind):
    """Page arrays of the cache, and what they hold."""
    return (k, v, k, v) if kind == "16" else filled(k, v, kind)


def attend(kind):
    return hmm.paged_attention if kind == "16" else hmm.paged_quant_attention


def with_zeros(k, v, table, gone):
    """The cache with a page of zeros behind it, and the table with `gone` entries there."""
    k0, v0 = (torch.cat([x.contiguous(), torch.zeros_like(x[:1])]) for x in (k, v))
    t = table.clone()
    for s, i in gone:
        t[s, i] = k.shape[0]
    return k0, v0, t


def left_behind(kind, seed, new, kv, hq, hk, d, pt, dtype, cuda):
    """A call of the same shape over a cache whose scale bytes are all 255, or whose values are
    large: what it leaves in shared memory."""
    q, k, v, table, cu, kv_len = make(cuda, seed, new, kv, hq, hk, d, pt, dtype, scale=5.0)
    kp, vp, _, _ = hold(k, 40 * v, kind)
    if kind != "16" and seed % 2:
        for pages in (kp, vp):
            raw(pages)[1].fill_(255)
    return lambda: attend(kind)(q, kp, vp, table, cu, kv_len)


SHAPES = [  # new, kv, hq, hk, d, pt, entries that are gone
    ([1] * 12, [300] * 12, 8, 2, 128, 16, [(0, 3), (1, 0), (2, 18), (3, 7), (3, 8)]),          # rows kernel
    ([1] * 12, [300] * 12, 8, 2, 64, 32, [(0, 3), (1, 0), (2, 9)]),
    ([1] * 12, [300] * 12, 2, 1, 256, 16, [(0, 3), (4, 18)]),
    ([2] * 5, [90] * 5, 6, 2, 128, 4, [(0, 3), (1, 21), (2, 22), (2, 0)]),
    ([40] * 6, [500] * 6, 8, 2, 128, 16, [(0, 3), (1, 0), (2, 31), (3, 29), (3, 30)]),         # chunk kernel
    ([40] * 6, [500] * 6, 8, 2, 64, 16, [(0, 3), (1, 0), (2, 31), (3, 29)]),
    ([40] * 6, [500] * 6, 4, 2, 256, 32, [(0, 3), (1, 0), (2, 15), (4, 13)]),
    ([130] * 3, [400] * 3, 4, 1, 96, 48, [(0, 0), (1, 8), (2, 3)]),
    ([200] * 2, [640] * 2, 4, 2, 128, 128, [(0, 0), (1, 4)]),
    ([50] * 4, [333] * 4, 8, 2, 128, 8, [(i, j) for i in range(2) for j in range(42)]),        # every page
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_its_own_rows_are_over_zeros(cuda, shape, dtype, kind):
    *case, gone = shape
    new, kv, hq, hk, d, pt = case
    q, k, v, table, cu, kv_len = make(cuda, 80, *case, DT[dtype])
    kp, vp, k, v = hold(k, v, kind)
    k0, v0, t0 = with_zeros(k, v, table, gone)
    ref = reference(q, k0, v0, t0, new, kv)
    bad = table.clone()
    for i, (s, p) in enumerate(gone):
        bad[s, p] = (-1, k.shape[0], 1 << 30, -(1 << 31))[i % 4]
    before = [left_behind(kind, seed, *case, DT[dtype], cuda) for seed in (81, 82)]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    outs = []
    for i in range(4):
        before[i % 2]()
        out, lse = attend(kind)(q, kp, vp, bad, cu, kv_len, return_lse=True, status=status.zero_())
        check(out, lse, ref)
        assert status.item() == 1
        outs.append((out, lse))
    for out, lse in outs[1:]:
        assert torch.equal(out, outs[0][0]) and torch.equal(lse, outs[0][1]), "the same call, the same bits"


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_of_a_widened_sequence(cuda, kind):
    new, kv, hq, hk, d, pt = [300, 3], [420, 100], 8, 2, 128, 16
    q, k, v, table, cu, kv_len = make(cuda, 83, new, kv, hq, hk, d, pt, torch.bfloat16)
    kp, vp, k, v = filled(k, v, kind)
    gone = [(0, 2), (0, 26), (1, 4)]
    k0, v0, t0 = with_zeros(k, v, table, gone)
    bad = long_table(table, pt, hk, hq, sum(new))
    for s, p in gone:
        bad[s, p] = -1
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = hmm.paged_quant_attention(q, kp, vp, bad, cu, kv_len, return_lse=True, status=status)
    check(out, lse, reference(q, k0, v0, t0, new, kv))
    assert status.item() == 1


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_seq,new", [(6, 1), (12, 8)])
def test_of_a_shared_prefix(cuda, kind, n_seq, new):
    """The pages of the prefix are those of the group's first row, for all its sequences; a
    tail's are its own."""
    hq, hk, d, pt, prefix = 8, 2, 128, 16, 320
    news, kv = [new] * n_seq, [prefix + 60] * n_seq
    q, k, v, table, cu, kv_len = make(cuda, 84, news, kv, hq, hk, d, pt, torch.bfloat16)
    table[1:, :prefix // pt] = table[0, :prefix // pt]
    kp, vp, k, v = hold(k, v, kind)
    gone = [(s, 5) for s in range(n_seq)] + [(2, prefix // pt + 1)]
    k0, v0, t0 = with_zeros(k, v, table, gone)
    bad = table.clone()
    bad[0, 5] = k.shape[0]
    bad[2, prefix // pt + 1] = -1
    cg, pl = groups_of([(0, n_seq, prefix)], n_seq, cuda)
    before = [left_behind(kind, seed, news, kv, hq, hk, d, pt, torch.bfloat16, cuda) for seed in (85, 86)]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    for i in range(2):
        before[i]()
        out, lse = hmm.paged_prefix_attention(q, kp, vp, bad, cu, kv_len, cg, pl, return_lse=True, status=status.zero_())
        check(out, lse, with_join(reference(q, k0, v0, t0, news, kv)))
        assert status.item() == 1

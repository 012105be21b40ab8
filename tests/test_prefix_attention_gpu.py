"""paged_prefix_attention against softmax attention in float64, each sequence by itself.

Tolerance: that of paged_attention (test_serve_attention_gpu.py), and for the join of the two
parts: their lse are rounded to fp32 and subtracted (2^-23 max |lse| each way), an exponential,
a division and two products (2^-20 together), which moves a part's share of the result by twice
as much; the parts' own results are fp32."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_BOUNDS, HmmError, set_wait_limit_ns
from heteromm_b200.paged import check_status
from test_quant_attention_gpu import filled, long_table, raw
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def ints(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def shared(cuda, seed, groups, new, kv, hq, hk, d, pt, dtype, pad=0, scale=1.0):
    """A batch as forks leave it.  groups: (first sequence, end, prefix).  Full pages of a prefix
    are the first sequence's with new tokens, a partly filled last one is copied."""
    q, k, v, table, cu, kv_len = make(cuda, seed, new, kv, hq, hk, d, pt, dtype, pad=pad, scale=scale)
    for a, b, n in groups:
        live = [s for s in range(a, b) if new[s] > 0]
        n = min([n] + [kv[s] - new[s] for s in live])
        if len(live) < 2 or n <= 0:
            continue
        for s in live[1:]:
            table[s, :n // pt] = table[live[0], :n // pt]
            if n % pt:
                src, dst = table[live[0], n // pt].item(), table[s, n // pt].item()
                k[dst, :, :n % pt], v[dst, :, :n % pt] = k[src, :, :n % pt], v[src, :, :n % pt]
    return q, k, v, table, cu, kv_len, groups_of(groups, len(new), cuda)


def groups_of(groups, n_seq, cuda):
    """cu_group and prefix_len: sequences between two groups form one without a prefix."""
    cu, prefix = [groups[0][0] if groups else 0], []
    for a, b, n in groups:
        if a > cu[-1]:
            cu.append(a)
            prefix.append(0)
        cu.append(b)
        prefix.append(n)
    return ints(cu, cuda), ints(prefix, cuda)


def with_join(ref):
    out, lse, tol, ltol = ref
    top = torch.where(torch.isfinite(lse), lse.abs(), 0.0)
    join = 2.0 ** -22 * top + 2.0 ** -20
    share = torch.where(torch.isfinite(out), out.abs(), 0.0)
    # (tol holds A = sum p |v| / sum p with a factor of eps / 2 at least, of the type: 2^-8 or 2^-11)
    return out, lse, tol + 2 * join[..., None] * (share + tol * 2.0 ** 11), ltol + join


BATCHES = [  # groups (first, end, prefix), new, kv, hq, hk, d, pt
    ([(0, 4, 777)], [1] * 4, [800, 778, 900, 1001], 32, 8, 128, 16),
    ([(0, 20, 2000)], [1] * 20, [2001 + 37 * i for i in range(20)], 16, 2, 128, 16),
    ([(0, 3, 64), (3, 9, 500), (9, 11, 1)], [2] * 11, [70, 66, 99] + [502 + i for i in range(6)] + [3, 200], 8, 2, 64, 16),
    ([(1, 5, 130)], [1, 3, 40, 1, 17, 1], [50, 140, 400, 131, 333, 9], 8, 2, 128, 16),       # some outside
    ([(0, 6, 300)], [1, 0, 2, 0, 1, 5], [301, 0, 400, 5, 320, 310], 4, 1, 96, 16),           # empty ones among them
    ([(0, 6, 300)], [0, 0, 2, 0, 1, 5], [0, 7, 400, 5, 320, 310], 4, 1, 64, 24),             # the first has no pages
    ([(0, 3, 190)], [1, 4, 1], [200, 150, 90], 4, 2, 64, 16),                               # a prefix cut by a sequence
    ([(0, 2, 100)], [50, 1], [50, 200], 4, 2, 64, 16),                                       # one that is all new
    ([(0, 1, 100), (1, 2, 50)], [1, 3], [200, 100], 4, 2, 64, 16),                           # alone: nothing shared
    ([(0, 40, 1111)], [3] * 40, [1114 + (53 * i) % 400 for i in range(40)], 7, 1, 128, 32),
    ([(0, 3, 250)], [130, 7, 300], [400, 300, 550], 8, 2, 64, 16),                           # chunks
    ([(0, 70, 600), (70, 75, 100)], [2] * 75, [610 + (7 * i) % 90 for i in range(70)] + [110] * 5, 4, 1, 128, 16),  # 560 rows
    ([(0, 9, 333)], [1] * 9, [340 + i for i in range(9)], 4, 2, 256, 16),
    ([(0, 5, 90)], [1] * 5, [100 + i for i in range(5)], 6, 2, 80, 5),                       # pages of the rows kernel alone
    ([(0, 2, 0)], [1, 1], [33, 20], 2, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("batch", BATCHES)
def test_formula(cuda, batch, dtype):
    groups, new, kv, hq, hk, d, pt = batch
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 40, groups, new, kv, hq, hk, d, pt, DT[dtype], pad=5)
    n = sum(new)
    out = torch.full((n + 5, hq, d), 9.0, dtype=DT[dtype], device=cuda)
    got, lse = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, out=out, return_lse=True, max_new=max(new))
    assert got is out and (out[n:] == 9.0).all()
    check(got, lse, with_join(reference(q, k, v, table, new, kv)))
    again, lse2 = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, return_lse=True)
    assert torch.equal(again[:n].view(torch.int16), got[:n].view(torch.int16)) and \
        torch.equal(lse2[:n].view(torch.int32), lse[:n].view(torch.int32)), "the same call, the same bits"
    got = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, scale=-0.07)
    check(got, None, with_join(reference(q, k, v, table, new, kv, scale=-0.07)))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("batch", [b for b in BATCHES if b[5] % 32 == 0 and b[6] * b[5] // 32 % 16 == 0])
def test_formula_in_8_bits(cuda, batch, dtype, kind):
    groups, new, kv, hq, hk, d, pt = batch
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 41, groups, new, kv, hq, hk, d, pt, DT[dtype], pad=2)
    kp, vp, k, v = filled(k, v, kind)
    got, lse = hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, return_lse=True)
    check(got, lse, with_join(reference(q, k, v, table, new, kv)))


@pytest.mark.parametrize("batch", [BATCHES[10], BATCHES[11], ([(1, 4, 300)], [5, 260, 20, 1, 200], [90, 600, 350, 301, 700], 8, 2, 128, 16)])
def test_widened_parts(cuda, batch):
    """Groups and tails of 512 rows and more, whose keys are widened first, beside others."""
    groups, new, kv, hq, hk, d, pt = batch
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 52, groups, new, kv, hq, hk, d, pt, torch.bfloat16)
    kp, vp, k, v = filled(k, v, "e4m3")
    wide = long_table(table, pt, hk, hq, max(sum(new), 256))
    got, lse = hmm.paged_prefix_attention(q, kp, vp, wide, cu, kv_len, cg, pl, return_lse=True)
    check(got, lse, with_join(reference(q, k, v, table, new, kv)))


def test_rows_of_nobody_before_the_first_sequence(cuda):
    groups, new, kv = [(0, 3, 64)], [1, 2, 1, 4], [80, 90, 66, 30]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 53, groups, new, kv, 8, 2, 128, 16, torch.bfloat16, pad=9)
    ref = with_join(reference(q[5:], k, v, table, new, kv))
    out = torch.full_like(q, 9.0)
    hmm.paged_prefix_attention(q, k, v, table, cu + 5, kv_len, cg, pl, out=out)
    check(out[5:], None, ref)
    assert (out[:5] == 9.0).all() and (out[5 + sum(new):] == 9.0).all()


def test_prefix_is_read_from_one_row(cuda):
    """The group's first sequence with new tokens names the prefix's pages: what the others' rows
    hold there does not reach a finite result."""
    groups, new, kv = [(0, 4, 160)], [1] * 4, [200, 170, 161, 300]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 42, groups, new, kv, 8, 2, 128, 16, torch.bfloat16)
    ref = reference(q, k, v, table, new, kv)
    table[1:, :10] = torch.arange(10, dtype=torch.int32, device=cuda)
    check(hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl), None, with_join(ref))


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("d,pt", [(128, 16), (64, 16), (80, 5)])
def test_values_that_are_not_finite(cuda, value, d, pt):
    """In slots behind the ends and pages of nobody they reach nothing; in the prefix every row
    of the group, in a tail its own; a bad key is NaN in every column."""
    groups, new, kv = [(0, 6, 200)], [1, 2, 1, 40, 1, 1], [260, 205, 201, 300, 230, 222]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 43, groups, new, kv, 8, 2, d, pt, torch.bfloat16)
    keep = torch.zeros((k.shape[0], pt), dtype=torch.bool, device=cuda)
    for s, L in enumerate(kv):
        for i in range(L):
            keep[table[s, i // pt].item(), i % pt] = True
    k.transpose(1, 2)[~keep] = value
    v.transpose(1, 2)[~keep] = value
    call = lambda: hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, return_lse=True)  # noqa: E731
    clean = lambda: reference(q, k, v, table, new, kv)  # noqa: E731
    out, lse = call()
    assert torch.isfinite(out).all()
    check(out, lse, with_join(clean()))
    for s, p in ((0, 240), (3, 290)):            # tails: in the middle of the fourth one's new tokens
        v[table[s, p // pt].item(), :, p % pt, 3] = value
    out, lse = call()
    check(out, lse, with_join(clean()))
    v[table[0, 70 // pt].item(), 1, 70 % pt, 5] = value          # the prefix: one head, one column
    out, lse = call()
    check(out, lse, with_join(clean()))
    if value != value:
        k[table[0, 30 // pt].item(), 0, 30 % pt, 0] = value
        out, lse = call()
        check(out, lse, with_join(clean()))
        assert torch.isnan(out[:, :4]).all() and torch.isnan(lse[:, :4]).all()


def test_a_bad_group_in_8_bits(cuda):
    groups, new, kv = [(0, 3, 100)], [1] * 3, [120, 101, 130]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 44, groups, new, kv, 4, 2, 64, 16, torch.bfloat16)
    kp, vp, k, v = filled(k, v, "int8")
    k, v = k.contiguous(), v.contiguous()
    for page, at in ((table[0, 3].item(), 5), (table[2, 7].item(), 10)):
        codes, scales = raw(vp)
        codes[page, :, at, 32:], scales[page, :, at, 1] = 0, 255
        v[page, :, at, 32:] = NAN
    out, lse = hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, return_lse=True)
    check(out, lse, with_join(reference(q, k, v, table, new, kv)))


def test_scores_far_apart(cuda):
    """One part outweighs the other by hundreds: its share is all."""
    groups, new, kv = [(0, 5, 400)], [1] * 5, [450 + i for i in range(5)]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 45, groups, new, kv, 4, 1, 64, 16, torch.bfloat16, scale=30.0)
    out, lse = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, return_lse=True)
    check(out, lse, with_join(reference(q, k, v, table, new, kv)))
    k[table[0, :400 // 16].long()] = -INF       # the prefix has no weight at all
    q = q.abs() + 0.1
    out, lse = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, return_lse=True)
    check(out, lse, with_join(reference(q, k, v, table, new, kv)))


def test_no_groups_is_the_plain_call(cuda):
    new, kv = [1, 30, 0], [100, 90, 4]
    q, k, v, table, cu, kv_len = make(cuda, 46, new, kv, 8, 2, 128, 16, torch.bfloat16)
    out, lse = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, ints([0], cuda), ints([], cuda), return_lse=True)
    check(out, lse, with_join(reference(q, k, v, table, new, kv)))
    none = hmm.paged_prefix_attention(q[:0], k, v, table, torch.zeros_like(cu), kv_len, ints([0], cuda), ints([], cuda))
    assert none.shape == (0, 8, 128)


def test_flags(cuda):
    groups, new, kv = [(0, 3, 100), (3, 5, 64)], [1] * 5, [120, 101, 130, 65, 80]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 47, groups, new, kv, 4, 2, 64, 16, torch.float16)
    ref = with_join(reference(q, k, v, table, new, kv))
    for bad_cg, bad_pl in (([0, 3, 6], [100, 64]), ([-1, 3, 5], [100, 64]), ([0, 3, 2], [100, 64]), ([0, 3, 5], [-1, 64]),
                           ([0, 3, 5], [100, 1 << 20])):
        with pytest.raises(HmmError) as e:
            hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, ints(bad_cg, cuda), ints(bad_pl, cuda))
        assert e.value.status == HMM_ERR_BOUNDS
    for lengths, offsets in (([120, 101, 4000, 65, 80], None), (None, [0, 1, 2, 1, 4, 5]), (None, [0, 1, 2, 3, 4, 6])):
        l2 = kv_len if lengths is None else ints(lengths, cuda)
        c2 = cu if offsets is None else ints(offsets, cuda)
        with pytest.raises(HmmError) as e:
            hmm.paged_prefix_attention(q, k, v, table, c2, l2, cg, pl)
        assert e.value.status == HMM_ERR_BOUNDS
    table[4, 1] = k.shape[0]                    # a page of a prefix, and only the fifth's row says so: not read
    check(hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl), None, ref)
    table[3, 1] = -1
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, status=status)
    with pytest.raises(HmmError):
        check_status(status)
    check(out[:3], None, tuple(x[:3] for x in ref))      # the other group's rows


def test_a_wait_that_runs_out_is_an_error(cuda):
    groups, new, kv = [(0, 30, 700)], [1] * 30, [720] * 30
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 48, groups, new, kv, 8, 2, 128, 16, torch.bfloat16)
    try:
        set_wait_limit_ns(0)
        with pytest.raises(HmmError, match="HMM_ERR_TIMEOUT"):
            hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl)
    finally:
        set_wait_limit_ns(-1)
    check(hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl), None, with_join(reference(q, k, v, table, new, kv)))


def test_captured_and_on_two_streams(cuda):
    """Two graphs of different batches replayed in turn while lengths and prefixes change, then
    both batches at once on streams of their own."""
    cases = []
    for seed, groups, new, kv, hq, hk, d in ((49, [(0, 12, 500)], [1] * 12, [560] * 12, 8, 2, 128), (50, [(0, 2, 90), (2, 5, 40)], [2] * 5, [140] * 5, 4, 1, 64)):
        q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, seed, groups, new, kv, hq, hk, d, 16, torch.bfloat16)
        status, out = torch.zeros(1, dtype=torch.int32, device=cuda), torch.empty_like(q)

        def call(q=q, k=k, v=v, table=table, cu=cu, kv_len=kv_len, cg=cg, pl=pl, out=out, status=status):
            return hmm.paged_prefix_attention(q, k, v, table, cu, kv_len, cg, pl, out=out, status=status)

        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        cases.append((g, call, new, kv, q, k, v, table, kv_len, pl, out, status))
    for i in range(3):
        for g, *_ in cases:
            g.replay()
        for _, _, new, kv, q, k, v, table, kv_len, pl, out, status in cases:
            check(out, None, with_join(reference(q, k, v, table, new, kv_len.tolist())))
            check_status(status)
            kv_len -= 7
            pl -= 11
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                c[1]()
    torch.cuda.synchronize()
    for _, _, new, kv, q, k, v, table, kv_len, pl, out, status in cases:
        check(out, None, with_join(reference(q, k, v, table, new, kv_len.tolist())))


@pytest.mark.parametrize("kind", [None, "e4m3"])
def test_a_served_conversation(cuda, kind):
    """A prompt, three forks of it, steps of all four behind the shared prefix: append, prefix
    attention and, for the same rows, the plain attention of the same cache."""
    hq, hk, d, pt, n_pages, n_seq = 8, 2, 64, 16, 64, 5
    g = torch.Generator(device=cuda).manual_seed(51)
    if kind:
        k_pages, v_pages = (hmm.quant_pages(n_pages, hk, pt, d, device=cuda) for _ in range(2))
        append, attend = hmm.paged_quant_append, hmm.paged_quant_attention
    else:
        k_pages = torch.full((n_pages, hk, pt, d), NAN, dtype=torch.bfloat16, device=cuda)
        v_pages = k_pages.clone()
        append, attend = hmm.paged_kv_append, hmm.paged_attention
    table = torch.full((n_seq, 12), -1, dtype=torch.int32, device=cuda)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=cuda)
    kv_len = torch.zeros(n_seq, dtype=torch.int32, device=cuda)
    rope = hmm.rope_table(256, d, device=cuda)
    cg, pl = ints([0, 4], cuda), ints([0], cuda)

    def step(new):
        nonlocal table, refs, kv_len
        q, k, v = torch.randn((sum(new), hq + 2 * hk, d), generator=g, device=cuda).to(torch.bfloat16).split([hq, hk, hk], dim=1)
        cu = ints([0] + list(np.cumsum(new)), cuda)
        table, refs, kv_len = hmm.paged_grow(table, refs, kv_len, ints(new, cuda), pt)
        q = append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope)
        out = hmm.paged_prefix_attention(q, k_pages, v_pages, table, cu, kv_len, cg, pl)
        plain = attend(q, k_pages, v_pages, table, cu, kv_len)
        kp, vp, kv = k_pages, v_pages, kv_len.tolist()
        if kind:
            every, c, l = (ints(x, cuda) for x in (list(range(n_pages)), [0, n_pages * pt], [n_pages * pt]))
            held = hmm.paged_quant_read(k_pages, v_pages, every[None], c, l, n_pages * pt)
            kp, vp = (x.reshape(n_pages, pt, hk, d).transpose(1, 2) for x in held)
        ref = reference(q, kp, vp, table, new, kv)
        check(plain, None, ref)
        check(out, None, with_join(ref))

    step([75, 0, 0, 0, 9])
    table, refs, kv_len = hmm.paged_fork(table, refs, kv_len, ints([0, 0, 0], cuda), ints([1, 2, 3], cuda), k_pages, v_pages)
    pl.fill_(75)
    step([1, 1, 1, 1, 1])
    step([3, 1, 20, 1, 0])
    table, refs, kv_len = hmm.paged_free(table, refs, kv_len, ints([0], cuda))
    table, refs, _ = hmm.paged_compact(table, refs, k_pages, v_pages)
    step([0, 1, 1, 2, 1])

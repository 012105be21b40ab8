"""paged_quant_attention against softmax attention in float64 over the values that the cache
holds, which are numbers of the queries' type: the tolerance is the one derived for
paged_attention over a cache of that type (test_serve_attention_gpu.py)."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_BOUNDS, HmmError, set_wait_limit_ns
from heteromm_b200.paged import check_status
from test_quant_cache_gpu import KIND
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def filled(k, v, kind):
    """Quantised page arrays of the same tokens, and what they hold in the type of k."""
    n, hk, pt, d = k.shape
    pages = [hmm.quant_pages(n, hk, pt, d, KIND[kind], k.device) for _ in range(2)]
    table = torch.arange(n, dtype=torch.int32, device=k.device)[None]
    cu, kv = (torch.tensor(x, dtype=torch.int32, device=k.device) for x in ([0, n * pt], [n * pt]))
    hmm.paged_quant_append(None, *(x.transpose(1, 2).reshape(n * pt, hk, d) for x in (k, v)), *pages, table, cu, kv)
    held = hmm.paged_quant_read(*pages, table, cu, kv, n * pt, dtype=k.dtype)
    return *pages, *(x.reshape(n, pt, hk, d).transpose(1, 2) for x in held)


def raw(pages):
    """(codes [n_pages, heads, page_tokens, D], scale bytes [..., D / 32]) of a page array: views."""
    n, h, t, row = pages.shape
    g = row // 33
    flat = pages.view(torch.uint8).view(n, h, t * row)
    return flat[..., :t * g * 32].unflatten(-1, (t, g * 32)), flat[..., t * g * 32:].unflatten(-1, (t, g))


def long_table(table, pt, hk, hq, tokens):
    """The table with empty columns behind it: a call that could come to so many products of chunks and
    long contexts that it widens the keys of those with 512 rows first."""
    columns = -(-4096 * 128 // (max(1, tokens * (hq // hk) // 256) * hk * pt)) + 1
    table = torch.nn.functional.pad(table, (0, columns), value=-1)
    size = hmm.load().hmm_paged_quant_attention_workspace_size
    assert size(table.shape[0], tokens, hq, hk, 64, table.shape[1] * pt, 0) > size(table.shape[0], tokens, hq, hk, 64, pt, 0) + (1 << 20)
    return table


def run_case(cuda, seed, new, kv, hq, hk, d, pt, dtype, kind, pad=0, max_new=0, kscale=1.0, wide=False, **kw):
    q, k, v, table, cu, kv_len = make(cuda, seed, new, kv, hq, hk, d, pt, DT[dtype], pad=pad, scale=kscale)
    kp, vp, k, v = filled(k, v, kind)
    if wide:
        table = long_table(table, pt, hk, hq, sum(new) + pad)
    out = torch.full((sum(new) + pad, hq, d), 9.0, dtype=DT[dtype], device=cuda)
    got, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, out=out, return_lse=True, max_new=max_new, **kw)
    assert got is out and (out[sum(new):] == 9.0).all()
    check(got, lse, reference(q, k, v, table, new, kv, **kw))
    again, lse2 = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, return_lse=True, max_new=max_new, **kw)
    n = sum(new)
    assert torch.equal(again[:n].view(torch.int16), got[:n].view(torch.int16)) and \
        torch.equal(lse2[:n].view(torch.int32), lse[:n].view(torch.int32)), "the same call, the same bits"


SHAPES = [  # new, kv, hq, hk, d, pt
    ([1], [1], 1, 1, 64, 16),
    ([1], [777], 32, 8, 128, 16),
    ([1, 1, 1, 1], [1, 16, 17, 4099], 8, 2, 128, 16),
    ([0, 1, 0, 3, 0], [5, 0, 0, 2, 9], 4, 2, 64, 8),
    ([5] * 6, [5, 6, 64, 65, 1000, 333], 28, 4, 128, 32),
    ([1, 130, 1, 33], [900, 130, 1, 300], 8, 2, 128, 16),
    ([300], [300], 6, 2, 64, 64),
    ([257, 3], [700, 3], 3, 3, 128, 128),
    ([100, 7], [129, 200], 14, 2, 96, 48),
    ([64, 2], [65, 2], 4, 1, 256, 16),
    ([70, 1], [1000, 501], 8, 8, 96, 16),
    ([40, 9], [77, 9], 6, 1, 128, 4),
    ([20, 1], [50, 33], 2, 1, 32, 16),
    ([129], [2100], 130, 1, 64, 16),
    ([31], [200], 160, 1, 32, 16),
    ([400, 1, 40], [500, 513, 40], 7, 1, 160, 16),
    ([3, 30], [77, 90], 6, 2, 256, 2),
    ([2, 17], [75, 300], 4, 2, 64, 24),
    ([1, 2, 20], [40, 300, 33], 4, 2, 192, 40),
]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_causal(cuda, shape, dtype, kind):
    run_case(cuda, 7, *shape, dtype, kind, pad=5)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 1), (128, 128), (129, 33), (5000, 4)])
def test_window(cuda, shape, window, sinks):
    run_case(cuda, 8, *shape, "bf16", "e4m3", window=window, sinks=sinks)


@pytest.mark.parametrize("shape", SHAPES)
def test_all_keys_and_scale(cuda, shape):
    run_case(cuda, 9, *shape, "fp16", "int8", causal=False, scale=0.3)
    run_case(cuda, 9, *shape, "bf16", "int8", scale=-0.05)
    run_case(cuda, 9, *shape, "fp16", "e4m3", scale=0.0)


@pytest.mark.parametrize("kind,dtype", [("e4m3", "bf16"), ("int8", "fp16")])
@pytest.mark.parametrize("shape", [
    ([600], [600], 2, 1, 64, 16),                                 # one sequence, widened whatever it holds
    ([0], [40], 4, 2, 64, 16),
    ([700, 1, 300, 3, 130], [900, 50, 301, 700, 2000], 8, 2, 128, 16),
    ([256, 200, 260], [300, 1000, 261], 2, 1, 128, 4),            # 512 rows, 400, 520; small pages
    ([520, 40], [530, 400], 3, 3, 96, 16),
    ([128, 128, 1], [128, 700, 9], 8, 2, 256, 2),
    ([600, 520, 3], [100, 530, 2], 4, 4, 64, 16),                 # fewer cached than new tokens
])
def test_chunks_of_many_rows(cuda, shape, kind, dtype):
    """Their keys are widened into the workspace first, beside sequences that are not."""
    run_case(cuda, 13, *shape, dtype, kind, pad=600, wide=True)
    run_case(cuda, 13, *shape, dtype, kind, pad=600, max_new=max(shape[0]), wide=max(shape[0]) * shape[2] // shape[3] >= 512,
             window=100, sinks=5)
    run_case(cuda, 13, *shape, dtype, kind, pad=600, wide=True, causal=False, scale=0.2)
    run_case(cuda, 13, *shape, dtype, kind, pad=3, scale=-0.1)


def test_widened_values_that_are_not_finite(cuda):
    """NaN groups in seen and unseen places of a chunk whose keys are widened, in a captured call."""
    new, kv, pt = [300, 1], [420, 50], 16
    q, k, v, table, cu, kv_len = make(cuda, 32, new, kv, 8, 2, 128, pt, torch.bfloat16)
    kp, vp, k, v = filled(k, v, "e4m3")
    k, v = k.contiguous(), v.contiguous()
    wide = long_table(table, pt, 2, 8, 301)
    for pages in (kp, vp):                       # behind the sequence's end
        codes, scales = raw(pages)
        codes[table[0, 419 // pt].item(), :, 420 % pt:] = 255
        scales[table[0, 419 // pt].item(), :, 420 % pt:] = 255
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    hmm.paged_quant_attention(q, kp, vp, wide, cu, kv_len, status=status)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = hmm.paged_quant_attention(q, kp, vp, wide, cu, kv_len, return_lse=True, status=status)
    g.replay()
    check(out, lse, reference(q, k, v, table, new, kv))
    for p in (380, 130):                         # seen by some rows, and by all
        page = table[0, p // pt].item()
        codes, scales = raw(vp)
        codes[page, 1, p % pt, 64:96], scales[page, 1, p % pt, 2] = 0, 255
        v[page, 1, p % pt, 64:96] = NAN
        g.replay()
        check(out, lse, reference(q, k, v, table, new, kv))
    check_status(status)
    wide[0, 3] = k.shape[0]
    g.replay()
    with pytest.raises(HmmError):
        check_status(status)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_queries_at_the_ends_of_bf16(cuda, kind):
    """Rows of 2^120 and of 2^-120, one large value beside small ones, rows of zeros: scores are
    those of the values."""
    new, kv = [1, 3, 20], [200, 90, 333]
    q, k, v, table, cu, kv_len = make(cuda, 33, new, kv, 4, 2, 64, 16, torch.bfloat16)
    q[0, 0] *= 2.0 ** -120
    q[1, 1] = 0
    q[2, 2, 7] = 2.0 ** 14
    q[5] *= 2.0 ** -30
    kp, vp, k, v = filled(k, v, kind)
    k = k.contiguous()
    out, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, return_lse=True)
    check(out, lse, reference(q, k, v, table, new, kv))
    big = q * 2.0 ** 110
    out, lse = hmm.paged_quant_attention(big, kp, vp, table, cu, kv_len, scale=2.0 ** -113, return_lse=True)
    check(out, lse, reference(big, k, v, table, new, kv, scale=2.0 ** -113))


def test_rows_of_nobody_before_the_first_sequence(cuda):
    new, kv = [2, 30, 1], [50, 400, 33]
    q, k, v, table, cu, kv_len = make(cuda, 34, new, kv, 8, 2, 128, 16, torch.float16, pad=7)
    kp, vp, k, v = filled(k, v, "int8")
    ref = reference(q[4:], k, v, table, new, kv)
    out = torch.full_like(q, 9.0)
    hmm.paged_quant_attention(q, kp, vp, table, cu + 4, kv_len, out=out)
    check(out[4:], None, ref)
    assert (out[:4] == 9.0).all() and (out[4 + sum(new):] == 9.0).all()
    k2, v2 = (torch.full((sum(new) + 7, 2, 128), 9.0, dtype=torch.float16, device=cuda) for _ in range(2))
    hmm.paged_quant_read(kp, vp, table, cu + 4, kv_len, sum(new) + 7, dtype=torch.float16, out=(k2, v2))
    assert (k2[:4] == 9.0).all() and (v2[4 + sum(new):] == 9.0).all()
    assert torch.equal(k2[4], k[table[0, 3].item(), :, 0]) and torch.equal(v2[36], v[table[2, 2].item(), :, 0])


def test_what_the_workspace_has_no_room_for(cuda):
    """64 KV heads of 256: room for 16,384 widened tokens, and three chunks over 8,000 each."""
    run_case(cuda, 14, [512, 530, 3, 515], [8000, 8100, 70, 8001], 64, 64, 256, 64, "bf16", "e4m3")


@pytest.mark.parametrize("max_new", [0, 1, 4, 1000])
def test_hint_is_only_a_hint(cuda, max_new):
    run_case(cuda, 10, [1, 50, 1, 4], [300, 50, 1000, 4], 8, 2, 128, 16, "bf16", "e4m3", max_new=max_new)


@pytest.mark.parametrize("dtype,kind", [("bf16", "e4m3"), ("fp16", "e4m3"), ("bf16", "int8"), ("fp16", "int8")])
def test_peaked_scores_and_ends_of_the_range(cuda, dtype, kind):
    """Scores far apart; values near the largest and below the smallest scale's step."""
    run_case(cuda, 11, [1, 200], [3000, 1500], 8, 2, 128, 16, dtype, kind, kscale=40.0)
    new, kv = [1, 40], [500, 300]
    q, k, v, table, cu, kv_len = make(cuda, 12, new, kv, 4, 2, 128, 16, DT[dtype])
    k[..., :32] *= 2.0 ** -20
    v[..., :32] *= 2.0 ** -20
    v[..., 32:64] *= 2.0 ** 11
    v[..., 64:96] *= 2.0 ** -12
    k[..., 96:] = 0
    kp, vp, k, v = filled(k, v, kind)
    out, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, return_lse=True)
    check(out, lse, reference(q, k, v, table, new, kv))


@pytest.mark.parametrize("d,pt,hq,hk", [(64, 16, 4, 2), (128, 16, 8, 2), (128, 64, 2, 2), (256, 16, 2, 1), (96, 16, 4, 2), (128, 4, 4, 2)])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_nothing_unseen_is_read(cuda, d, pt, hq, hk, kind):
    """Scale bytes of 255 and codes of all ones in the slots behind a sequence's end, in pages of
    nobody, in tokens behind the window, in pages that are gone (-1), and in tokens that only
    later rows see: the rows that do not see them are as if they were not there."""
    new, kv = [150, 1, 6], [400, 333, 90]
    for window, sinks in ((0, 0), (40, 3)):
        q, k, v, table, cu, kv_len = make(cuda, 14, new, kv, hq, hk, d, pt, torch.bfloat16)
        kp, vp, k, v = filled(k, v, kind)
        k, v = k.contiguous(), v.contiguous()
        keep = torch.zeros((k.shape[0], pt), dtype=torch.bool, device=cuda)
        for s, (n, L) in enumerate(zip(new, kv)):
            first = max(0, L - n - window + 1) if window else 0
            for i in list(range(min(sinks, L))) + list(range(first, L)):
                keep[table[s, i // pt].item(), i % pt] = True
        for pages in (kp, vp):
            codes, scales = raw(pages)
            codes.transpose(1, 2)[~keep] = 255
            scales.transpose(1, 2)[~keep] = 255
        if window:
            for s, (n, L) in enumerate(zip(new, kv)):
                first = max(0, L - n - window + 1)
                for i in range(-(-sinks // pt), first // pt):
                    table[s, i] = -1 if i % 2 else 1 << 30
        ts = table.clamp(-1, k.shape[0] - 1)
        out, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, window=window, sinks=sinks, return_lse=True)
        check(out, lse, reference(q, k, v, ts, new, kv, window=window, sinks=sinks))
        # a late token of the first and the third sequence: a group of its values is NaN
        for s, p in ((0, 399 - 20), (2, 88)):
            page = table[s, p // pt].item()
            codes, scales = raw(vp)
            scales[page, :, p % pt, 1] = 255
            codes[page, :, p % pt, 32:64] = 0
            v[page, :, p % pt, 32:64] = NAN
        page = table[0, 390 // pt].item()
        codes, scales = raw(kp)
        scales[page, :, 390 % pt, 0] = 255
        codes[page, :, 390 % pt, :32] = 0
        k[page, :, 390 % pt, :32] = NAN
        out = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, window=window, sinks=sinks)
        check(out, None, reference(q, k, v, ts, new, kv, window=window, sinks=sinks))


@pytest.mark.parametrize("batch", [([1, 1, 1, 1], [1, 17, 50, 64], 8, 2, 128, 16), ([1, 1, 3], [33, 4000, 97], 16, 8, 64, 16),
                                   ([40, 1, 130], [50, 1, 900], 8, 2, 128, 16), ([300], [333], 16, 4, 64, 64)])
def test_queries_that_are_not_finite(cuda, batch):
    new, kv = batch[:2]
    q, k, v, table, cu, kv_len = make(cuda, 60, *batch, torch.float16)
    kp, vp, k, v = filled(k, v, "e4m3")
    first = 0
    for n in new:
        q[first + n - 1, -1, 3] = NAN
        q[first, 0, 5] = INF
        first += n
    ref = reference(q, k, v, table, new, kv)
    assert torch.isnan(ref[0]).any()
    out, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, return_lse=True)
    check(out, lse, ref)


def test_the_result_is_that_of_the_16_bit_cache(cuda):
    """The same kernel family over the values in 16 bits: as near as two orders of sums are."""
    new, kv = [1, 40, 1], [900, 333, 50]
    q, k, v, table, cu, kv_len = make(cuda, 30, new, kv, 8, 2, 128, 16, torch.bfloat16)
    kp, vp, k, v = filled(k, v, "int8")
    ref = reference(q, k, v, table, new, kv)
    a = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len)
    b = hmm.paged_attention(q, k.contiguous(), v.contiguous(), table, cu, kv_len)
    assert not ((a.double() - b.double()).abs() > 2 * ref[2]).any()


@pytest.mark.parametrize("layout", ["interleaved", "qkv", "bits", "one head"])
def test_layouts(cuda, layout):
    new, kv, hq, hk, d, pt = [1, 40], [100, 61], 4, 2, 64, 16
    if layout == "one head":
        hq = hk = 1
    q, k, v, table, cu, kv_len = make(cuda, 16, new, kv, hq, hk, d, pt, torch.bfloat16)
    kp, vp, k, v = filled(k, v, "e4m3")
    ref = reference(q, k, v, table, new, kv)
    if layout == "interleaved":
        both = torch.stack([kp.view(torch.uint8), vp.view(torch.uint8)], 1).view(torch.float8_e4m3fn)
        kp, vp = both[:, 0], both[:, 1]
    elif layout == "qkv":
        wide = torch.full((41, hq + 2 * hk, d + 8), NAN, dtype=torch.bfloat16, device=cuda)
        wide[:, 1:1 + hq, :d] = q
        q = wide[:, 1:1 + hq, :d]
    elif layout == "bits":
        q = q.view(torch.int16)
    elif layout == "one head":
        kp, vp = kp[:, 0], vp[:, 0]
    out = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len)
    check(out.view(torch.bfloat16), None, ref)


def test_flags(cuda):
    new, kv = [2, 30, 1, 1], [40, 60, 16, 20]
    q, k, v, table, cu, kv_len = make(cuda, 17, new, kv, 4, 2, 64, 16, torch.float16)
    kp, vp, k, v = filled(k, v, "int8")
    ref = reference(q, k, v, table, new, kv)
    bad = table.clone()
    bad[0, 1] = k.shape[0]
    bad[1, 0] = -1
    with pytest.raises(HmmError) as e:
        hmm.paged_quant_attention(q, kp, vp, bad, cu, kv_len)
    assert e.value.status == HMM_ERR_BOUNDS
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = hmm.paged_quant_attention(q, kp, vp, bad, cu, kv_len, status=status)
    check(out[32:], None, tuple(x[32:] for x in ref))      # the other sequences' rows
    with pytest.raises(HmmError):
        check_status(status)
    for lengths, offsets in (([40, 60, 16, 65], None), ([-1, 60, 16, 20], None), (None, [0, 2, 32, 33, 35]),
                             (None, [0, 2, 1, 33, 34]), (None, [-1, 2, 32, 33, 34])):
        l2 = kv_len if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda)
        c2 = cu if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=cuda)
        with pytest.raises(HmmError) as e:
            hmm.paged_quant_attention(q, kp, vp, table, c2, l2)
        assert e.value.status == HMM_ERR_BOUNDS


def test_a_wait_that_runs_out_is_an_error(cuda):
    q, k, v, table, cu, kv_len = make(cuda, 31, [1, 200], [900, 500], 8, 2, 128, 16, torch.bfloat16)
    kp, vp, k, v = filled(k, v, "e4m3")
    try:
        set_wait_limit_ns(0)
        with pytest.raises(HmmError, match="HMM_ERR_TIMEOUT"):
            hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len)
    finally:
        set_wait_limit_ns(-1)
    out = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len)
    check(out, None, reference(q, k, v, table, [1, 200], [900, 500]))


def test_far_pages(cuda):
    """A cache of more than 2^32 bytes a side: offsets pass 32 bits."""
    pt, d, hk = 64, 128, 4
    n_pages = (5 << 30) // (pt * (d + 4) * hk)
    pages = [hmm.quant_pages(n_pages, hk, pt, d, torch.int8, cuda) for _ in range(2)]
    for new in ([1, 1], [1, 90]):
        kv = [100, 150]
        q, k, v, ts, cu, kv_len = make(cuda, 22, new, kv, 8, hk, d, pt, torch.bfloat16, spare=0)
        kp, vp, k, v = filled(k, v, "int8")
        far = torch.tensor([n_pages - 1 - 3 * i for i in range(k.shape[0])], device=cuda)
        pages[0][far], pages[1][far] = kp, vp
        table = torch.where(ts >= 0, far[ts.long().clamp(min=0)].to(torch.int32), -1)
        out = hmm.paged_quant_attention(q, *pages, table, cu, kv_len)
        check(out, None, reference(q, k, v, ts, new, kv))


def test_a_captured_served_step(cuda):
    """Append and attention in one graph, replayed while the lengths grow; two graphs of
    different batches replayed in turn."""
    hq, hk, d, pt = 8, 2, 128, 16
    graphs = []
    for seed, n_seq, n in ((18, 3, 1), (19, 2, 20)):
        kv = [200 + 31 * i for i in range(n_seq)]
        q, k, v, table, cu, _ = make(cuda, seed, [n] * n_seq, [x + 8 * n for x in kv], hq, hk, d, pt, torch.bfloat16)
        kp, vp, _, _ = filled(k, v, "e4m3")
        kv_len = torch.tensor(kv, dtype=torch.int32, device=cuda)
        kn, vn = (torch.randn((n * n_seq, hk, d), device=cuda).to(torch.bfloat16) for _ in range(2))
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = torch.empty_like(q)

        def step(q=q, kp=kp, vp=vp, table=table, cu=cu, kv_len=kv_len, kn=kn, vn=vn, out=out, status=status, n=n):
            kv_len += n
            hmm.paged_quant_append(None, kn, vn, kp, vp, table, cu, kv_len, status=status)
            hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, max_new=n, out=out, status=status)

        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append((g, [n] * n_seq, [x + n for x in kv], q, kp, vp, table, out, status, step))   # step keeps its tensors
    for i in range(3):
        for g, *_ in graphs:
            g.replay()
        for _, new, kv, q, kp, vp, table, out, status, _ in graphs:
            now = [x + (i + 1) * new[0] for x in kv]
            n, hk_, t, row = kp.shape
            every = torch.arange(n, dtype=torch.int32, device=cuda)[None]
            c, l = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, n * t], [n * t]))
            held = hmm.paged_quant_read(kp, vp, every, c, l, n * t)
            k, v = (x.reshape(n, t, hk_, -1).transpose(1, 2) for x in held)
            check(out, None, reference(q, k, v, table, new, now))
            check_status(status)


def test_two_streams_at_once(cuda):
    """Two calls of different batches on two streams share nothing."""
    cases = []
    for seed, new, kv in ((20, [1] * 8, [3000] * 8), (21, [200], [2500])):
        q, k, v, *rest = make(cuda, seed, new, kv, 8, 2, 128, 16, torch.bfloat16)
        kp, vp, k, v = filled(k, v, "e4m3")
        cases.append(((q, kp, vp, *rest), reference(q, k, v, rest[0], new, kv), torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(10):
        for t, _, st, outs in cases:
            with torch.cuda.stream(st):
                outs.append(hmm.paged_quant_attention(*t, status=torch.zeros(1, dtype=torch.int32, device=cuda)))
    torch.cuda.synchronize()
    for _, ref, _, outs in cases:
        for o in outs:
            check(o, None, ref)

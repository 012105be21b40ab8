"""paged_attention where scores are not finite: a NaN in a query or in keys that a row
sees is NaN in its result, in both kernels, whole units and joined pieces alike."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")

BATCHES = [  # new, kv, hq, hk, d, pt
    ([1, 1, 1, 1], [1, 17, 50, 64], 8, 2, 128, 16),       # rows kernel: a CTA has all of a unit
    ([1, 1, 3], [33, 4000, 97], 16, 8, 64, 16),           # pieces of several CTAs
    ([1], [2049], 4, 1, 256, 16),
    ([5, 1], [700, 65], 6, 2, 80, 5),                     # pages that only the rows kernel takes, joined
    ([40, 1, 130], [50, 1, 900], 8, 2, 128, 16),          # both kernels, the chunk kernel's units cut
    ([300], [333], 16, 4, 64, 64),
    ([2600, 700], [2600, 2049], 16, 8, 128, 16),          # whole units
]


def poison(kind, q, k, table, new, kv, pt):
    """NaN scores of some rows of every sequence; returns nothing, changes q or k."""
    first = 0
    for s, (n, L) in enumerate(zip(new, kv)):
        if kind == "a query":                     # one head of the last token
            q[first + n - 1, -1, 3] = NAN
        elif kind == "all queries":
            q[first:first + n] = NAN
        elif kind == "all keys":
            k[table[s, :-(-L // pt)].long()] = NAN
        elif kind == "a page":
            k[table[s, (L - 1) // pt // 2].item()] = NAN
        elif kind == "16 keys":                   # a warp's share of a tile, whatever the page size
            for p in range(16, min(32, L)):
                k[table[s, p // pt].item(), :, p % pt] = NAN
        elif kind == "newest key":
            k[table[s, (L - 1) // pt].item(), :, (L - 1) % pt, 0] = NAN
        elif kind == "inf - inf":                 # keys that overflowed: products of both signs
            k[table[s, (L - 1) // pt].item(), 0, (L - 1) % pt] = INF
        first += n


@pytest.mark.parametrize("kind", ["a query", "all queries", "all keys", "a page", "16 keys", "newest key", "inf - inf"])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_nan_scores(cuda, batch, kind, dtype):
    new, kv = batch[:2]
    q, k, v, table, cu, kv_len = make(cuda, 60, *batch, DT[dtype])
    poison(kind, q, k, table, new, kv, batch[5])
    ref = reference(q, k, v, table, new, kv)
    assert torch.isnan(ref[0]).any()
    out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True)
    check(out, lse, ref)
    assert torch.equal(torch.isnan(lse).double(), torch.isnan(ref[1]).double())
    hint = hmm.paged_attention(q, k, v, table, cu, kv_len, max_new=1)        # the rows kernel, however many rows
    check(hint, None, ref)


@pytest.mark.parametrize("at", [0, 15, 16, 48, 63, 64, 1000])
@pytest.mark.parametrize("window", [0, 20])
def test_a_nan_key_at_any_place_of_a_tile(cuda, at, window):
    """The newest key, which is the only one that a warp sees at the start of its 16 keys."""
    batch = ([1, 2, 40], [at + 1, at + 2, at + 40], 8, 2, 128, 16)
    new, kv = batch[:2]
    q, k, v, table, cu, kv_len = make(cuda, 61, *batch, torch.bfloat16)
    for s in range(3):
        k[table[s, at // 16].item(), :, at % 16] = NAN
    kw = dict(window=window, sinks=3 if window else 0)
    ref = reference(q, k, v, table, new, kv, **kw)
    out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True, **kw)
    check(out, lse, ref)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()


def test_infinite_scores_of_few_rows(cuda):
    """+inf is NaN, -inf a weight of zero, only -inf zeros: the rows kernel as the formula."""
    new, kv, d = [1, 1, 1, 2], [100, 40, 2000, 33], 64
    q, k, v, table, cu, kv_len = make(cuda, 62, new, kv, 2, 1, d, 16, torch.bfloat16)
    q = q.abs() + 0.1
    k[table[0, 3].item(), 0, 5] = INF
    k[table[1, :3].long()] = -INF
    k[table[2, 100].item()] = -INF
    k[table[3, :2].long()] = -INF
    ref = reference(q, k, v, table, new, kv)
    out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True)
    check(out, lse, ref)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert (out[1] == 0).all() and (lse[1] == -np.inf).all() and torch.isfinite(out[2]).all()


def put(t, table, s, p, pt, col, value):
    t[table[s, p // pt].item(), :, p % pt, col] = value


@pytest.mark.parametrize("kind", ["first nan", "first inf", "inf in the middle", "inf of both signs", "inf and nan", "newest inf",
                                  "many inf", "many nan", "not seen by all"])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("dtype,window", [("bf16", 0), ("fp16", 0), ("bf16", 40)])
def test_values_that_are_not_finite(cuda, batch, kind, dtype, window):
    """Rows that see them have what the formula gives, the others are as if they were not there."""
    new, kv, pt = batch[0], batch[1], batch[5]
    q, k, v, table, cu, kv_len = make(cuda, 63, *batch, DT[dtype])
    d = v.shape[-1]
    for s, (n, L) in enumerate(zip(new, kv)):
        if kind == "first nan":
            put(v, table, s, 0, pt, 5, NAN)
        elif kind == "first inf":
            put(v, table, s, 0, pt, 5, INF)
            put(v, table, s, 0, pt, d - 1, -INF)
        elif kind == "inf in the middle":
            put(v, table, s, L // 2, pt, 0, INF)
        elif kind == "inf of both signs":
            put(v, table, s, 0, pt, 1, INF)
            put(v, table, s, L - 1, pt, 1, -INF)
            put(v, table, s, L // 2, pt, 2, -INF)
        elif kind == "inf and nan":
            put(v, table, s, L // 3, pt, 7, INF)
            put(v, table, s, 2 * L // 3, pt, 7, NAN)
        elif kind == "newest inf":
            put(v, table, s, L - 1, pt, 3, INF)
        elif kind in ("many inf", "many nan"):
            for p in range(L // 2, L // 2 + min(5, L - L // 2)):
                v[table[s, p // pt].item(), :, p % pt] = INF if kind == "many inf" else NAN
        else:                                     # seen by the second half of the new tokens
            put(v, table, s, L - n // 2 - 1, pt, 4, INF)
            put(v, table, s, L - n // 2 - 1, pt, 6, NAN)
    kw = dict(window=window, sinks=2 if window else 0)
    ref = reference(q, k, v, table, new, kv, **kw)
    for hint in (0, 1):
        out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True, max_new=hint, **kw)
        check(out, lse, ref)
        inf = torch.isinf(ref[0])
        assert torch.equal(out.double()[inf], ref[0][inf])


@pytest.mark.parametrize("scale", [0.0, 1e-30])
def test_a_scale_of_nothing(cuda, scale):
    """All seen keys weigh the same, whatever their scores; the rows that see none are zeros."""
    for batch in BATCHES:
        new, kv = batch[:2]
        q, k, v, table, cu, kv_len = make(cuda, 64, *batch, torch.bfloat16)
        kw = dict(scale=scale, window=50, sinks=1)
        out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True, **kw)
        check(out, lse, reference(q, k, v, table, new, kv, **kw))


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("what", ["k", "v", "q", "late v"])
def test_one_bad_value_costs_little(cuda, value, what):
    """A NaN or infinity that a long prompt's rows see does not send them through their keys one
    after another: 227 ms when it did, and 0.15 ms without it."""
    n, pt = 4096, 16
    q, k, v, table, cu, kv_len = make(cuda, 65, [n], [n], 32, 8, 128, pt, torch.bfloat16)
    if what == "q":
        q[:, :, 0] = value
    elif what == "late v":
        put(v, table, 0, n // 2, pt, 9, value)
    else:
        put(k if what == "k" else v, table, 0, 0, pt, 9, value)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    times = []
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        hmm.paged_attention(q, k, v, table, cu, kv_len, status=status)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    assert min(times) < 10, times


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("new", [1, 3, 40, 300])
@pytest.mark.parametrize("low", [40, 120, 600])
def test_an_infinity_behind_a_small_weight(cuda, dtype, new, low):
    """exp(-low) may be nothing in the weights' type or in fp32; it is above zero all the same.
    Only a score of -inf has no weight: its product with an infinity is NaN."""
    L, d, pt = 900, 64, 16
    q, k, v, table, cu, kv_len = make(cuda, 66, [new], [L], 2, 1, d, pt, DT[dtype])
    q[:] = 0
    q[..., 0] = 1
    k.clamp_(-2, 2)
    ids = table[0].long()
    for p, col, x in ((5, 1, INF), (300, 2, -INF), (L - new, 3, INF), (299, 4, INF), (500, 4, -INF)):
        k[ids[p // pt], 0, p % pt, 0] = -low
        put(v, table, 0, p, pt, col, x)
    ref = reference(q, k, v, table, [new], [L], scale=1.0)
    for hint in (0, 1):
        out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, scale=1.0, return_lse=True, max_new=hint)
        check(out, lse, ref)
        inf = torch.isinf(ref[0])
        assert inf[..., 1:4].all() and torch.isnan(ref[0][..., 4]).all() and torch.equal(out.double()[inf], ref[0][inf])
    k[ids[0], 0, 5, 0] = -INF
    out = hmm.paged_attention(q, k, v, table, cu, kv_len, scale=1.0)
    check(out, None, reference(q, k, v, table, [new], [L], scale=1.0))
    assert torch.isnan(out[..., 1]).all()

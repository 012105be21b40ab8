"""paged_attention against softmax attention in float64.

Tolerance, from the arithmetic the entry point states.  With A = sum_i p_i |v_i| / sum_i
p_i: the weights are rounded to the cache's type (half a step, eps / 2 of A) and the result
is (eps / 2 of its value); an fp32 score is off by at most delta = (D + 8) 2^-23 B + 2^-22
max |s| + 2^-20, B = max_i |scale| sum_d |q_d k_id| (D products, a 24-bit sum that may
truncate, the scaling, the exponential), which moves a weight's share by 2 delta; fp32 sums
of n weights over pieces by 2^-18.  A weight below the type's smallest normal number (fp16) loses
at most finfo.tiny * eps of the largest: n of them, of sum 1 or more, n tiny eps max |v|."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_BOUNDS, HmmError
from heteromm_b200.paged import check_status

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(cuda, seed, new, kv, hq, hk, d, pt, dtype, spare=3, pad=0, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    counts = [-(-x // pt) for x in kv]
    n_pages = sum(counts) + spare
    k = (scale * torch.randn((n_pages, hk, pt, d), generator=g, device=cuda)).to(dtype)
    v = torch.randn((n_pages, hk, pt, d), generator=g, device=cuda).to(dtype)
    perm = torch.randperm(n_pages, generator=g, device=cuda).to(torch.int32).cpu()
    table = torch.full((len(new), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = perm[at:at + c]
        at += c
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    q = torch.randn((sum(new) + pad, hq, d), generator=g, device=cuda).to(dtype)
    return q, k, v, table.to(cuda), cu.to(cuda), torch.tensor(kv, dtype=torch.int32, device=cuda)


def reference(q, k, v, table, new, kv, causal=True, window=0, sinks=0, scale=None):
    """Per token and head in float64: (out, lse, tolerance of out, tolerance of lse).
    Values that a row does not see are left out of its sums, not multiplied by zero."""
    hq, d = q.shape[1:]
    hk, pt = k.shape[1], k.shape[2]
    g = hq // hk
    fi = torch.finfo(q.dtype)
    scale = d ** -0.5 if scale is None else scale
    total = sum(new)
    out = torch.zeros((total, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((total, hq), -np.inf, dtype=torch.float64, device=q.device)
    ltol = torch.zeros_like(lse)
    at = 0
    for s, (n, L) in enumerate(zip(new, kv)):
        if n == 0:
            continue
        if L > 0:
            ids = table[s, :-(-L // pt)].long().clamp(min=0)
            pos = torch.arange(L - n, L, device=q.device)[:, None]
            key = torch.arange(L, device=q.device)[None, :]
            see = (key <= pos) if causal else torch.ones((n, L), dtype=torch.bool, device=q.device)
            if window:
                see = see & ((key > pos - window) | (key < sinks))
            for h in range(hk):
                kk = k[ids, h].reshape(-1, d)[:L].double()
                vv = v[ids, h].reshape(-1, d)[:L].double()
                for j in range(g):
                    qq = q[at:at + n, h * g + j].double()
                    x = torch.where(see, scale * (qq @ kk.T), -np.inf)
                    m = x.amax(-1, keepdim=True)
                    m = torch.where(m == -np.inf, 0.0, m)
                    p = torch.where(see, (x - m).exp(), 0.0)
                    z = p.sum(-1, keepdim=True)
                    # finite values by a product, the others added where they are seen
                    bad = ~torch.isfinite(vv)
                    num = p @ torch.where(bad, 0.0, vv)
                    for i in bad.any(-1).nonzero().flatten().tolist():
                        rows = see[:, i]
                        num[rows] += p[rows, i:i + 1] * torch.where(bad[i], vv[i], 0.0)
                    o = torch.where(z > 0, num / z, 0.0) if not torch.isnan(z).any() else torch.where(z == 0, 0.0, num / z)
                    mag = (p @ torch.where(bad, 0.0, vv).abs()) / z.clamp(min=1e-300)
                    b = abs(scale) * torch.where(see, qq.abs() @ torch.where(torch.isfinite(kk), kk, 0.0).abs().T, 0.0).amax(-1, keepdim=True)
                    top = torch.where(see & torch.isfinite(x), x, 0.0).abs().amax(-1, keepdim=True)
                    delta = (d + 8) * 2.0 ** -23 * b + 2.0 ** -22 * top + 2.0 ** -20
                    out[at:at + n, h * g + j] = o
                    tol[at:at + n, h * g + j] = fi.eps / 2 * (1 + fi.eps) * (o.abs() + mag) + (2 * delta + 2.0 ** -18) * mag + \
                        fi.tiny * fi.eps * (1 + L * torch.where(bad, 0.0, vv).abs().max())
                    lse[at:at + n, h * g + j] = (m + z.log()).squeeze(-1)
                    ltol[at:at + n, h * g + j] = (delta + 2.0 ** -18 + 2.0 ** -22 * top).squeeze(-1)
        at += n
    return out, lse, tol, ltol


def check(got, glse, ref):
    out, lse, tol, ltol = ref
    n = out.shape[0]
    got = got[:n].double()
    fin = torch.isfinite(out)
    assert torch.equal(torch.isfinite(got), fin), "what is finite"
    assert torch.equal(torch.isnan(got), torch.isnan(out)), "what is NaN"
    worst = ((got - out).abs() / tol.clamp(min=1e-30))[fin]
    assert worst.numel() == 0 or float(worst.max()) <= 1, float(worst.max())
    if glse is not None:
        glse = glse[:n].double()
        fin = torch.isfinite(lse)
        assert torch.equal(torch.isfinite(glse), fin)
        assert torch.equal(glse == -np.inf, lse == -np.inf)
        assert not ((glse - lse).abs() > ltol)[fin].any(), float((glse - lse).abs()[fin].max())


def run_case(cuda, seed, new, kv, hq, hk, d, pt, dtype, pad=0, max_new=0, kscale=1.0, **kw):
    q, k, v, table, cu, kv_len = make(cuda, seed, new, kv, hq, hk, d, pt, DT[dtype], pad=pad, scale=kscale)
    out = torch.full((sum(new) + pad, hq, d), 9.0, dtype=DT[dtype], device=cuda)
    got, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, out=out, return_lse=True, max_new=max_new, **kw)
    assert got is out and (out[sum(new):] == 9.0).all()
    check(got, lse, reference(q, k, v, table, new, kv, **kw))
    again, lse2 = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True, max_new=max_new, **kw)
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
    ([100, 7], [129, 200], 14, 2, 80, 24),
    ([64, 2], [65, 2], 4, 1, 256, 16),
    ([70, 1], [1000, 501], 8, 8, 96, 8),
    ([40, 9], [77, 9], 6, 1, 72, 5),
    ([20, 1], [50, 33], 2, 1, 8, 1),
    ([129], [2100], 130, 1, 64, 16),
    ([31], [200], 160, 1, 32, 16),
    ([400, 1, 40], [500, 513, 40], 7, 1, 136, 40),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_causal(cuda, shape, dtype):
    run_case(cuda, 7, *shape, dtype, pad=5)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 1), (128, 128), (129, 33), (5000, 4)])
def test_window(cuda, shape, window, sinks):
    run_case(cuda, 8, *shape, "bf16", window=window, sinks=sinks)


@pytest.mark.parametrize("shape", SHAPES)
def test_all_keys_and_scale(cuda, shape):
    run_case(cuda, 9, *shape, "fp16", causal=False, scale=0.3)
    run_case(cuda, 9, *shape, "bf16", scale=-0.05)


@pytest.mark.parametrize("max_new", [0, 1, 4, 1000])
def test_hint_is_only_a_hint(cuda, max_new):
    run_case(cuda, 10, [1, 50, 1, 4], [300, 50, 1000, 4], 8, 2, 128, 16, "bf16", max_new=max_new)


def test_peaked_scores(cuda):
    """Scores far apart: the running maximum moves by hundreds."""
    run_case(cuda, 11, [1, 200], [3000, 1500], 8, 2, 128, 16, "bf16", kscale=40.0)
    run_case(cuda, 12, [1, 200], [3000, 1500], 8, 2, 64, 16, "fp16", kscale=40.0)


def test_rising_scores(cuda):
    """Each key scores above all earlier ones: every tile moves the maximum."""
    new, kv, d = [3, 260], [2000, 900], 64
    q, k, v, table, cu, kv_len = make(cuda, 13, new, kv, 2, 1, d, 16, torch.bfloat16)
    q = torch.ones_like(q)
    for s, L in enumerate(kv):
        ramp = torch.linspace(-4, 4, L, device=cuda).to(torch.bfloat16)
        for i in range(-(-L // 16)):
            part = ramp[16 * i:16 * i + 16]
            k[table[s, i].item(), 0, :len(part)] = part[:, None]
    out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True)
    check(out, lse, reference(q, k, v, table, new, kv))


@pytest.mark.parametrize("d,pt,hq,hk", [(64, 16, 4, 2), (128, 16, 8, 2), (128, 64, 2, 2), (256, 16, 2, 1), (80, 5, 4, 2)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_nothing_unseen_is_read(cuda, d, pt, hq, hk, value):
    """NaN and infinities in the slots behind a sequence's end, in pages of nobody, in
    tokens behind the window, in pages that are gone (-1), and in tokens that only later
    rows see: the rows that do not see them are as if they were not there."""
    new, kv = [150, 1, 6], [400, 333, 90]
    for window, sinks in ((0, 0), (40, 3)):
        q, k, v, table, cu, kv_len = make(cuda, 14, new, kv, hq, hk, d, pt, torch.bfloat16)
        keep = torch.zeros((k.shape[0], pt), dtype=torch.bool, device=cuda)
        for s, (n, L) in enumerate(zip(new, kv)):
            first = max(0, L - n - window + 1) if window else 0
            for i in list(range(min(sinks, L))) + list(range(first, L)):
                keep[table[s, i // pt].item(), i % pt] = True
        k.transpose(1, 2)[~keep] = value
        v.transpose(1, 2)[~keep] = value
        if window:
            for s, (n, L) in enumerate(zip(new, kv)):
                first = max(0, L - n - window + 1)
                for i in range(-(-sinks // pt), first // pt):
                    table[s, i] = -1 if i % 2 else 1 << 30
        out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, window=window, sinks=sinks, return_lse=True)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        ks, vs = torch.where(torch.isfinite(k), k, 0), torch.where(torch.isfinite(v), v, 0)
        ts = table.clamp(-1, k.shape[0] - 1)
        check(out, lse, reference(q, ks, vs, ts, new, kv, window=window, sinks=sinks))
        # a late token of the first and the third sequence
        for s, p in ((0, 399 - 20), (2, 88)):
            v[table[s, p // pt].item(), :, p % pt, 1] = value
            vs[table[s, p // pt].item(), :, p % pt, 1] = value
        k[table[0, 390 // pt].item(), :, 390 % pt] = float("nan")
        ks[table[0, 390 // pt].item(), :, 390 % pt] = float("nan")
        out = hmm.paged_attention(q, k, v, table, cu, kv_len, window=window, sinks=sinks)
        check(out, None, reference(q, ks, vs, ts, new, kv, window=window, sinks=sinks))


def test_infinite_scores(cuda):
    """Keys of -inf (weights of zero), a row whose every score is -inf, one with +inf."""
    new, kv, d = [4, 200], [100, 300], 64
    q, k, v, table, cu, kv_len = make(cuda, 15, new, kv, 2, 1, d, 16, torch.bfloat16)
    q = q.abs() + 0.1
    for p in (0, 5, 50, 96):
        k[table[0, p // 16].item(), 0, p % 16] = -float("inf")
    for i in range(-(-300 // 16)):
        k[table[1, i].item()] = -float("inf")
    k[table[1, 18].item(), 0, 10] = 1.0      # position 298: the last two rows see it
    out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, return_lse=True)
    check(out, lse, reference(q, k, v, table, new, kv))
    assert (out[4:202] == 0).all() and (lse[4:202] == -float("inf")).all()
    k[table[0, 2].item(), 0, 3] = float("inf")
    out = hmm.paged_attention(q, k, v, table, cu, kv_len)
    assert torch.isnan(out[:4]).all() and torch.isfinite(out[4:]).all()


@pytest.mark.parametrize("kind", ["token-major", "interleaved", "qkv", "bits", "one head"])
def test_layouts(cuda, kind):
    new, kv, hq, hk, d, pt = [1, 40], [100, 61], 4, 2, 64, 16
    if kind == "one head":
        hq = hk = 1
    q, k, v, table, cu, kv_len = make(cuda, 16, new, kv, hq, hk, d, pt, torch.bfloat16)
    ref = reference(q, k, v, table, new, kv)
    if kind == "token-major":
        k, v = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    elif kind == "interleaved":
        both = torch.stack([k, v], 1)
        k, v = both[:, 0], both[:, 1]
    elif kind == "qkv":
        wide = torch.full((41, hq + 2 * hk, d + 8), float("nan"), dtype=torch.bfloat16, device=cuda)
        wide[:, 1:1 + hq, :d] = q
        q = wide[:, 1:1 + hq, :d]
    elif kind == "bits":
        q, k, v = q.view(torch.int16), k.view(torch.int16), v.view(torch.int16)
    elif kind == "one head":
        k, v = k[:, 0], v[:, 0]
    out = hmm.paged_attention(q, k, v, table, cu, kv_len)
    check(out.view(torch.bfloat16), None, ref)


def test_flags(cuda):
    new, kv = [2, 30, 1, 1], [40, 60, 16, 20]
    q, k, v, table, cu, kv_len = make(cuda, 17, new, kv, 4, 2, 64, 16, torch.float16)
    ref = reference(q, k, v, table, new, kv)
    bad = table.clone()
    bad[0, 1] = k.shape[0]
    bad[1, 0] = -1
    with pytest.raises(HmmError) as e:
        hmm.paged_attention(q, k, v, bad, cu, kv_len)
    assert e.value.status == HMM_ERR_BOUNDS
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = hmm.paged_attention(q, k, v, bad, cu, kv_len, status=status)
    check(out[32:], None, tuple(x[32:] for x in ref))      # the other sequences' rows
    with pytest.raises(HmmError):
        check_status(status)
    for lengths, offsets in (([40, 60, 16, 65], None), ([-1, 60, 16, 20], None), (None, [0, 2, 32, 33, 35]),
                             (None, [0, 2, 1, 33, 34]), (None, [-1, 2, 32, 33, 34])):
        l2 = kv_len if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda)
        c2 = cu if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=cuda)
        with pytest.raises(HmmError) as e:
            hmm.paged_attention(q, k, v, table, c2, l2)
        assert e.value.status == HMM_ERR_BOUNDS


def test_captured_step_with_moving_lengths(cuda):
    """One captured step of append and attention, replayed while the lengths grow; two
    graphs of different batches replayed in turn."""
    hq, hk, d, pt = 8, 2, 128, 16
    graphs = []
    for seed, n_seq, n in ((18, 3, 1), (19, 2, 20)):
        kv = [200 + 31 * i for i in range(n_seq)]
        cap = [x + 8 * n for x in kv]
        q, k, v, table, cu, _ = make(cuda, seed, [n] * n_seq, cap, hq, hk, d, pt, torch.bfloat16)
        kv_len = torch.tensor(kv, dtype=torch.int32, device=cuda)
        kn, vn = (torch.randn((n * n_seq, hk, d), device=cuda).to(torch.bfloat16) for _ in range(2))
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = torch.empty_like(q)

        def step(q=q, k=k, v=v, table=table, cu=cu, kv_len=kv_len, kn=kn, vn=vn, out=out, status=status, n=n):
            kv_len += n
            hmm.paged_kv_append(None, kn, vn, k, v, table, cu, kv_len, status=status)
            hmm.paged_attention(q, k, v, table, cu, kv_len, max_new=n, out=out, status=status)

        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append((g, [n] * n_seq, [x + n for x in kv], q, k, v, table, out, status, step))   # step keeps its tensors
    for i in range(3):
        for g, *_ in graphs:
            g.replay()
        for _, new, kv, q, k, v, table, out, status, _ in graphs:
            now = [x + (i + 1) * new[0] for x in kv]
            check(out, None, reference(q, k, v, table, new, now))
            check_status(status)


def test_two_streams_at_once(cuda):
    """Two calls of different batches on two streams share nothing."""
    cases = []
    for seed, new, kv in ((20, [1] * 8, [3000] * 8), (21, [200], [2500])):
        t = make(cuda, seed, new, kv, 8, 2, 128, 16, torch.bfloat16)
        cases.append((t, reference(t[0], t[1], t[2], t[3], new, kv), torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(10):
        for t, _, st, outs in cases:
            with torch.cuda.stream(st):
                outs.append(hmm.paged_attention(*t, status=torch.zeros(1, dtype=torch.int32, device=cuda)))
    torch.cuda.synchronize()
    for _, ref, _, outs in cases:
        for o in outs:
            check(o, None, ref)


def test_far_pages(cuda):
    """A cache of more than 2^32 bytes a side: offsets pass 32 bits."""
    pt, d, hk = 64, 128, 4
    n_pages = (5 << 30) // (pt * d * hk * 2)
    k = torch.zeros((n_pages, hk, pt, d), dtype=torch.bfloat16, device=cuda)
    v = torch.zeros((n_pages, hk, pt, d), dtype=torch.bfloat16, device=cuda)
    for new in ([1, 1], [1, 90]):
        kv = [100, 150]
        q, ks, vs, ts, cu, kv_len = make(cuda, 22, new, kv, 8, hk, d, pt, torch.bfloat16, spare=0)
        far = torch.tensor([n_pages - 1 - 3 * i for i in range(ks.shape[0])], device=cuda)
        k[far], v[far] = ks, vs
        table = torch.where(ts >= 0, far[ts.long().clamp(min=0)].to(torch.int32), -1)
        out = hmm.paged_attention(q, k, v, table, cu, kv_len)
        check(out, None, reference(q, ks, vs, ts, new, kv))
        new_k = torch.randn((sum(new), hk, d), device=cuda).to(torch.bfloat16)
        hmm.paged_kv_append(None, new_k, new_k, k, v, table, cu, kv_len)
        assert torch.equal(k[table[0, 1].item(), :, 99 - 64], new_k[0])


def test_a_served_conversation(cuda):
    """Grow, append, attend, fork, append differently, attend, free, compact, attend: the
    calls together, against attention over the plain history of each sequence."""
    hq, hk, d, pt, n_pages, n_seq = 8, 2, 64, 16, 64, 4
    dt = torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(23)
    k_pages = torch.full((n_pages, hk, pt, d), float("nan"), dtype=dt, device=cuda)
    v_pages = k_pages.clone()
    table = torch.full((n_seq, 12), -1, dtype=torch.int32, device=cuda)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=cuda)
    kv_len = torch.zeros(n_seq, dtype=torch.int32, device=cuda)
    rope = hmm.rope_table(256, d, device=cuda)
    history = [([], []) for _ in range(n_seq)]      # rotated keys and values as stored

    def step(new):
        nonlocal table, refs, kv_len
        total = sum(new)
        qkv = torch.randn((total, hq + 2 * hk, d), generator=g, device=cuda).to(dt)
        q, k, v = qkv.split([hq, hk, hk], dim=1)
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=cuda)
        table, refs, kv_len = hmm.paged_grow(table, refs, kv_len, torch.tensor(new, dtype=torch.int32, device=cuda), pt)
        qr = hmm.paged_kv_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope)
        out = hmm.paged_attention(qr, k_pages, v_pages, table, cu, kv_len)
        # the plain history: the same rotation through a cache of its own
        at = 0
        for s, n in enumerate(new):
            have = len(history[s][0])
            plain = torch.zeros((n + have, hk, 1, d), dtype=dt, device=cuda)
            pv = plain.clone()
            if n:
                hmm.paged_kv_append(None, k[at:at + n], v[at:at + n], plain, pv,
                                    torch.arange(n + have, dtype=torch.int32, device=cuda)[None],
                                    torch.tensor([0, n], dtype=torch.int32, device=cuda),
                                    torch.tensor([n + have], dtype=torch.int32, device=cuda), rope)
            history[s][0].extend(plain[have:, :, 0].unbind(0))
            history[s][1].extend(pv[have:, :, 0].unbind(0))
            at += n
        at = 0
        for s, n in enumerate(new):
            if n:
                hk_, hv_ = torch.stack(history[s][0])[:, :, None], torch.stack(history[s][1])[:, :, None]
                ids = torch.arange(len(history[s][0]), dtype=torch.int32, device=cuda)[None]
                ref = reference(qr[at:at + n], hk_, hv_, ids, [n], [len(history[s][0])])
                check(out[at:at + n], None, ref)
            at += n
        assert kv_len.tolist() == [len(h[0]) for h in history]

    step([37, 0, 5, 0])
    step([1, 16, 1, 0])
    table, refs, kv_len = hmm.paged_fork(table, refs, kv_len, torch.tensor([0], dtype=torch.int32, device=cuda),
                                         torch.tensor([3], dtype=torch.int32, device=cuda), k_pages, v_pages)
    history[3] = (list(history[0][0]), list(history[0][1]))
    step([1, 1, 0, 20])
    table, refs, kv_len = hmm.paged_free(table, refs, kv_len, torch.tensor([0, 2], dtype=torch.int32, device=cuda))
    history[0], history[2] = ([], []), ([], [])
    table, refs, live = hmm.paged_compact(table, refs, k_pages, v_pages)
    assert live.item() == int((refs > 0).sum()) and (refs[live.item():] == 0).all()
    step([0, 3, 40, 1])

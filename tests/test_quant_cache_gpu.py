"""A paged cache held in 8 bits: filling it (paged_quant_append) and reading it back
(paged_quant_read) against the format's definition in float64.

Values are stored as they come, so their codes are compared bit by bit.  Keys are normed and
turned in fp32, off by less than 2^-19 (|a| + |b|) (11 additions and a root in the norm, 4
products and roundings, 3 in the rotation, 2^-24 each), and rounded once, by at most half a
step of the code's grid with the scale that was stored; the scale is the least that holds the
group's largest key, or its neighbour where that lies within 2^-18 of the border.  Reading
back is exact."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_BOUNDS, HmmError
from heteromm_b200.paged import check_status
from test_serve_append_gpu import close, reference

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
KIND = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST = {"e4m3": 448.0, "int8": 127.0}
LOW = {"e4m3": -15, "int8": -22}
GRID = np.array([(1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) if b >> 3 else (b & 7) / 8 * 2.0 ** -6 for b in range(127)])


def decoded(pages, kind):
    """float64 [n_pages, heads, page_tokens, D] and the scale bytes, from the raw bytes, on the host."""
    n, h, t, row = pages.shape
    g = row // 33
    raw = pages.contiguous().view(torch.uint8).cpu().numpy().reshape(n, h, t * row)
    codes, s = raw[..., :t * g * 32].reshape(n, h, t, g, 32), raw[..., t * g * 32:].reshape(n, h, t, g)
    if kind == "int8":
        v = codes.view(np.int8).astype(np.float64)
    else:
        v = np.where(codes >= 128, -1.0, 1.0) * np.append(GRID, np.nan)[codes & 127]
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
    return (v * scale[..., None]).reshape(n, h, t, g * 32), s


def least_scale(x, kind):
    """Exponents of the groups of x [..., D] (float64): the least that hold them."""
    top = np.abs(x).reshape(*x.shape[:-1], -1, 32).max(-1)
    e = np.full(top.shape, 7)
    for p in range(6, LOW[kind] - 1, -1):
        e = np.where(top <= MOST[kind] * 2.0 ** p, p, e)
    return e


def stored(x, kind):
    """What x (float64, finite) is stored as."""
    e = least_scale(x, kind)
    z = np.clip(x.reshape(*e.shape, 32) / np.ldexp(1.0, e)[..., None], -MOST[kind], MOST[kind])
    step = 1.0 if kind == "int8" else np.ldexp(1.0, np.frexp(np.maximum(np.abs(z), 2.0 ** -6))[1] - 4)
    return (np.rint(z / step) * step * np.ldexp(1.0, e)[..., None]).reshape(x.shape)


def layout(new, kv, pt, hk, d, kind, cuda, seed, spare=2):
    """A cache of random bytes, a shuffled page table and the batch's vectors."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    counts = [-(-x // pt) for x in kv]
    n_pages = sum(counts) + spare
    pages = [torch.randint(0, 127, (n_pages, hk, pt, d + d // 32), generator=g, device=cuda, dtype=torch.uint8).view(KIND[kind])
             for _ in range(2)]
    perm = torch.randperm(n_pages, generator=g, device=cuda).to(torch.int32).cpu()
    table = torch.full((len(new), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = perm[at:at + c]
        at += c
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    return *pages, table.to(cuda), cu.to(cuda), torch.tensor(kv, dtype=torch.int32, device=cuda)


def places(new, kv, pt, table):
    seq = np.repeat(np.arange(len(new)), new)
    pos = np.concatenate([np.arange(x - n, x) for n, x in zip(new, kv)]).astype(np.int64)
    return table.cpu().numpy()[seq, pos // pt], pos % pt, pos


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,pt,rotary,interleaved,norm", [
    (128, 16, 128, False, True), (128, 4, 64, True, True), (128, 16, 36, False, False), (64, 8, 64, False, True),
    (32, 16, 32, False, True), (32, 16, 0, False, False), (96, 16, 96, False, True), (96, 48, 20, True, False),
    (256, 2, 256, False, True), (256, 16, 100, False, True), (160, 16, 160, False, True), (64, 24, 16, False, False)])
def test_append_and_read_formula(cuda, kind, dtype, d, pt, rotary, interleaved, norm):
    new, kv, hq, hk = [1, 0, 5, 19], [1, 7, 33, 20], 6, 3
    dt = DT[dtype]
    k_pages, v_pages, table, cu, kv_len = layout(new, kv, pt, hk, d, kind, cuda, 11 + d)
    total = sum(new)
    g = torch.Generator(device=cuda).manual_seed(d)
    qkv = (3 * torch.randn((total + 4, hq + 2 * hk, d), generator=g, device=cuda)).to(dt)   # 4 rows of padding
    q, k, v = qkv.split([hq, hk, hk], dim=1)
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g, device=cuda)).to(dt) if norm else None for _ in range(2))
    rope = hmm.rope_table(64, rotary, 500.0, cuda) if rotary else None
    out = torch.full((total + 4, hq, d), 7.0, dtype=dt, device=cuda)
    before = [x.clone() for x in (k_pages, v_pages)]
    r = hmm.paged_quant_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope, q_weight=wq, k_weight=wk, eps=1e-5,
                               interleaved=interleaved, out=out)
    assert r is out
    assert (out[total:] == 7.0).all()          # rows that no sequence owns
    phys, row, pos = places(new, kv, pt, table)
    rows = rope[torch.from_numpy(pos).to(cuda)] if rotary else None
    ref, mag = reference(q[:total], wq, rows, interleaved, 1e-5)
    close(out[:total], ref, mag, "q")
    got_k, s = (x[phys, :, row] for x in decoded(k_pages, kind))
    got_v = decoded(v_pages, kind)[0][phys, :, row]
    assert np.array_equal(got_v, stored(v[:total].double().cpu().numpy(), kind))
    ref, mag = (x.cpu().numpy() for x in reference(k[:total], wk, rows, interleaved, 1e-5))
    e = s.astype(np.int64) - 127
    assert (e >= least_scale(ref * (1 - 2.0 ** -18), kind)).all() and (e <= least_scale(ref * (1 + 2.0 ** -18), kind)).all()
    scale = np.repeat(np.ldexp(1.0, e), 32, -1)
    half = scale / 2 if kind == "int8" else np.maximum(np.abs(ref) * 2.0 ** -4, scale * 2.0 ** -10)
    assert (np.abs(got_k - ref) <= half * (1 + 2.0 ** -10) + 2.0 ** -18 * mag).all()
    # every other slot as it was, byte for byte
    for x, y in zip((k_pages, v_pages), before):
        x, y = decoded(x, kind), decoded(y, kind)
        mask = np.ones((x[0].shape[0], pt), dtype=bool)
        mask[phys, row] = False
        for a, b in zip(x, y):
            assert np.array_equal(a.swapaxes(1, 2)[mask], b.swapaxes(1, 2)[mask], equal_nan=True)
    # read back, in every type, rows of nobody left alone
    for t in DT.values():
        k2, v2 = (torch.full((total + 4, hk, d), 7.0, dtype=t, device=cuda) for _ in range(2))
        r = hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, total + 4, dtype=t, out=(k2, v2))
        assert r[0] is k2 and r[1] is v2
        assert (k2[total:] == 7.0).all() and (v2[total:] == 7.0).all()
        assert np.array_equal(k2[:total].double().cpu().numpy(), got_k)
        assert np.array_equal(v2[:total].double().cpu().numpy(), got_v)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_every_code_and_scale_reads_back(cuda, kind):
    """All codes with all scales that an append writes, in every type: exact."""
    pt, d, groups = 16, 128, 40
    pages = hmm.quant_pages(10, 3, pt, d, KIND[kind], cuda)
    assert pages.dtype == KIND[kind] and tuple(pages.shape) == (10, 3, pt, d + 4)
    raw = pages.view(torch.uint8).view(10, 3, -1)
    g = torch.Generator(device=cuda).manual_seed(3)
    codes = torch.randint(0, 256, (10, 3, pt * d), generator=g, device=cuda)
    codes[0, 0, :256] = torch.arange(256, device=cuda)
    codes = torch.where((codes & 127) == 127, 0, codes) if kind == "e4m3" else torch.where(codes == 128, 0, codes)
    raw[..., :pt * d] = codes.to(torch.uint8)
    raw[..., pt * d:] = torch.randint(127 + LOW[kind], 127 + 8, (10, 3, pt * 4), generator=g, device=cuda).to(torch.uint8)
    other = pages.flip(0)
    table = torch.arange(10, dtype=torch.int32, device=cuda)[None]
    n = 10 * pt
    cu, kv_len = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, n], [n]))
    for t in DT.values():
        k, v = hmm.paged_quant_read(pages, other, table, cu, kv_len, n, dtype=t)
        for got, p in ((k, pages), (v, other)):
            want = decoded(p, kind)[0].swapaxes(1, 2).reshape(n, 3, d)
            assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_groups_of_zeros_and_the_ends_of_the_range(cuda, kind):
    """Zeros, the smallest numbers, values beyond the largest (cut), infinities and NaN (the
    group reads as NaN, its neighbours do not), borders between scales."""
    pt, d, hk = 16, 128, 2
    m, low = MOST[kind], LOW[kind]
    x = torch.zeros((6, hk, d), device=cuda)
    x[0, 0, :] = -0.0
    x[0, 1, 5], x[0, 1, 40], x[0, 1, 127] = 2.0 ** -126, -2.0 ** -30, 2.0 ** -14
    x[1, 0, 3], x[1, 0, 4], x[1, 0, 33], x[1, 0, 70] = float("inf"), 1.0, 2.0, -3.0
    x[1, 1, 127], x[1, 1, 0] = float("nan"), 5.0
    x[2, 0, 0], x[2, 0, 1], x[2, 1, 31] = 3e38, -2.0, -3e38
    for i, f in enumerate((1.0, 1.0 + 2.0 ** -7, 1.0 - 2.0 ** -8, 0.5)):     # about the border between two scales
        x[3, 0, 32 * i] = m * f
        x[3, 0, 32 * i + 1] = -1.0
        x[3, 1, 32 * i] = -m * f * 2.0 ** low
    x[4] = torch.linspace(-m, m, d, device=cuda)
    x[5] = torch.linspace(-1, 1, d, device=cuda) * m * 2.0 ** (low - 3)
    x = x.to(torch.bfloat16)
    k_pages, v_pages = (hmm.quant_pages(2, hk, pt, d, KIND[kind], cuda) for _ in range(2))
    table = torch.tensor([[1]], dtype=torch.int32, device=cuda)
    cu, kv_len = (torch.tensor(y, dtype=torch.int32, device=cuda) for y in ([0, 6], [6]))
    assert hmm.paged_quant_append(None, x, x, k_pages, v_pages, table, cu, kv_len) is None
    k, v = hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, 6)
    ref = x.double().cpu().numpy()
    groups = ref.reshape(6, hk, 4, 32)
    bad = ~np.isfinite(groups).all(-1, keepdims=True) & np.ones_like(groups, dtype=bool)
    want = stored(np.where(bad, 0.0, groups).reshape(ref.shape), kind)
    want[bad.reshape(ref.shape)] = np.nan
    for got in (k, v):
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want[1, 0, :32]).all() and not np.isnan(want[1, 0, 32:]).any()
    assert want[2, 0, 0] == m * 128
    # fresh pages are zeros
    table[0, 0] = 0
    k, v = hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, 6, dtype=torch.float16)
    assert (k == 0).all() and (v == 0).all()


def test_whole_cache_read_and_empty_sequences(cuda):
    """Ragged lengths, none and one among them; token runs of one head; nothing to read."""
    kv, pt, d = [0, 1, 130, 0, 16, 17], 16, 64
    k_pages, v_pages, table, cu, kv_len = layout(kv, kv, pt, 1, d, "int8", cuda, 9)
    n = sum(kv)
    k, v = hmm.paged_quant_read(k_pages[:, 0], v_pages[:, 0], table, cu, kv_len, n, dtype=torch.float32)
    phys, row, _ = places(kv, kv, pt, table)
    assert np.array_equal(k.cpu().numpy(), decoded(k_pages, "int8")[0].astype(np.float32)[phys, :, row])
    assert np.array_equal(v.cpu().numpy(), decoded(v_pages, "int8")[0].astype(np.float32)[phys, :, row])
    none = torch.zeros(1, dtype=torch.int32, device=cuda)
    k, v = hmm.paged_quant_read(k_pages, v_pages, table[:0], none, none[:0], 0)
    assert k.shape == (0, 1, d)


def test_interleaved_pages_bits_and_in_place(cuda):
    """K and V pages in one array, heads of a wider block, bf16 bits as int16, q in place."""
    n_pages, pt, hk, hq, d = 9, 4, 2, 4, 128
    both = torch.zeros((n_pages, 2, hk + 1, pt, d + 4), dtype=torch.int8, device=cuda)
    k_pages, v_pages = both[:, 0, :hk], both[:, 1, 1:]
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn((6, hq + 2 * hk, d), generator=g, device=cuda).to(torch.bfloat16)
    q, k, v = x.clone().view(torch.int16).split([hq, hk, hk], dim=1)
    table = torch.tensor([[8, 0, 3]], dtype=torch.int32, device=cuda)
    cu, kv_len = (torch.tensor(y, dtype=torch.int32, device=cuda) for y in ([0, 6], [10]))
    rope = hmm.rope_table(16, 128, 10000.0, cuda)
    assert hmm.paged_quant_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope, out=q) is q
    ref, mag = reference(x, None, rope[4:10], False, 0.0)
    close(q.view(torch.bfloat16), ref[:, :hq], mag[:, :hq], "q")
    got = decoded(v_pages.contiguous(), "int8")[0]
    for i, p in enumerate(range(4, 10)):
        assert np.array_equal(got[int(table[0, p // pt]), :, p % pt],
                              stored(x[i, hq + hk:].double().cpu().numpy(), "int8"))
    assert (both[:, 0, hk] == 0).all() and (both[:, 1, 0] == 0).all()


def test_flags(cuda):
    """A bad page, a length beyond the table, a sequence longer than its cache, a cu that
    descends: flagged and skipped by both calls, the others done."""
    d, pt, hk = 64, 8, 1
    new, kv = [2, 1, 1, 3, 1], [12, 8, 3, 2, 99]
    k_pages, v_pages, table, cu, _ = layout(new, [12, 8, 3, 4, 8], pt, hk, d, "e4m3", cuda, 3)
    kv_len = torch.tensor(kv, dtype=torch.int32, device=cuda)
    table[0, 1] = k_pages.shape[0]
    table[1, 0] = -1
    k = torch.randn((8, hk, d), device=cuda).to(torch.float16)
    before = decoded(v_pages, "e4m3")[0]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    hmm.paged_quant_append(None, k, k, k_pages, v_pages, table, cu, kv_len, status=status)
    with pytest.raises(HmmError) as e:
        check_status(status)
    assert e.value.status == HMM_ERR_BOUNDS and status.item() == 1 | 16
    changed = np.argwhere((decoded(v_pages, "e4m3")[0] != before).any(-1).any(1)).tolist()
    # sequence 2's token; sequence 3 has two of its three tokens at positions 0 and 1
    assert sorted(changed) == sorted([[int(table[2, 0]), 2], [int(table[3, 0]), 0], [int(table[3, 0]), 1]])
    status.zero_()
    out = tuple(torch.full((8, hk, d), 7.0, dtype=torch.float32, device=cuda) for _ in range(2))
    hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, 8, dtype=torch.float32, out=out, status=status)
    assert status.item() == 1 | 16
    want = stored(k.double().cpu().numpy(), "e4m3")
    for x in out:
        x = x.cpu().numpy()
        assert np.array_equal(x[[3, 5, 6]], want[[3, 5, 6]])
        assert (x[[0, 1, 2, 4, 7]] == 7.0).all()
    cu[2] = 0
    with pytest.raises(HmmError) as e:
        hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, 8)
    assert e.value.status == HMM_ERR_BOUNDS


def test_pages_move_as_any_others(cuda):
    """Copy, fork, grow and compact on pages of 8 bits: the tokens read back the same."""
    n_pages, hk, pt, d = 12, 2, 16, 64
    g = torch.Generator(device=cuda).manual_seed(4)
    pages = [torch.randint(0, 127, (2, n_pages, hk, pt, d + 2), generator=g, device=cuda, dtype=torch.uint8).view(torch.float8_e4m3fn)
             for _ in range(2)]
    table = torch.tensor([[7, 3, -1], [-1, -1, -1], [9, -1, -1]], dtype=torch.int32, device=cuda)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=cuda)
    refs[[7, 3, 9]] = 1
    kv_len = torch.tensor([20, 0, 5], dtype=torch.int32, device=cuda)

    def tokens(layer, s, n):
        cu, kv = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, n], [n]))
        return hmm.paged_quant_read(pages[0][layer], pages[1][layer], table[s:s + 1].contiguous(), cu, kv, n, dtype=torch.float32)

    want = [tokens(layer, s, n) for layer in range(2) for s, n in ((0, 20), (2, 5))]
    one = torch.tensor([0], dtype=torch.int32, device=cuda)
    table, refs, kv_len = hmm.paged_fork(table, refs, kv_len, one, one + 1, *pages)
    assert kv_len.tolist() == [20, 20, 5] and table[1, 0] == 7 and table[1, 1] == 0
    forked = [tokens(layer, 1, 20) for layer in range(2)]
    table, refs, kv_len = hmm.paged_free(table, refs, kv_len, one)
    table, refs, live = hmm.paged_compact(table, refs, *pages)
    assert live.item() == 3
    moved = [tokens(layer, s, n) for layer in range(2) for s, n in ((1, 20), (2, 5))]
    hmm.paged_copy_pages(*pages, table[2, :1].contiguous(), one + 11)
    table[2, 0] = 11
    copied = [tokens(layer, 2, 5) for layer in range(2)]
    for a, b in ((forked[0], want[0]), (forked[1], want[2]), (copied[0], want[1]), (copied[1], want[3])):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for a, b in zip(moved, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_many_sequences_stream_and_graph(cuda):
    """Every sequence of a large ragged batch finds its rows; on a stream of its own; captured
    and replayed with other lengths."""
    rng = np.random.RandomState(0)
    new = rng.randint(0, 4, 1500).tolist()
    kv = [n + int(x) for n, x in zip(new, rng.randint(0, 30, 1500))]
    d, pt, hk = 32, 16, 1
    k_pages, v_pages, table, cu, kv_len = layout(new, [x + 3 for x in kv], pt, hk, d, "int8", cuda, 4)
    kv_len.copy_(torch.tensor(kv, dtype=torch.int32))
    total = sum(new)
    x = torch.randn((total, hk, d), device=cuda).to(torch.bfloat16)
    want = stored(x.double().cpu().numpy(), "int8")
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        hmm.paged_quant_append(None, x, x, k_pages, v_pages, table, cu, kv_len)
        k, v = hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, total, status=status)
    torch.cuda.current_stream().wait_stream(st)
    assert np.array_equal(k.double().cpu().numpy(), want) and np.array_equal(v.double().cpu().numpy(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hmm.paged_quant_append(None, x, x, k_pages, v_pages, table, cu, kv_len, status=status)
        k, v = hmm.paged_quant_read(k_pages, v_pages, table, cu, kv_len, total, status=status)
    kv_len += 3
    x.copy_(torch.randn((total, hk, d), device=cuda))
    graph.replay()
    want = stored(x.double().cpu().numpy(), "int8")
    assert status.item() == 0
    assert np.array_equal(k.double().cpu().numpy(), want) and np.array_equal(v.double().cpu().numpy(), want)


def test_offsets_past_31_bits(cuda):
    """A page array of more than 2^32 bytes: its last page is the one that is filled and read."""
    n_pages, hk, pt, d = 70000, 8, 64, 128
    pages = torch.zeros((n_pages, hk, pt, d + 4), dtype=torch.int8, device=cuda)   # 4.7 GB
    table = torch.tensor([[n_pages - 1]], dtype=torch.int32, device=cuda)
    cu, kv_len = (torch.tensor(y, dtype=torch.int32, device=cuda) for y in ([0, 3], [64]))
    x = torch.randn((3, hk, d), device=cuda).to(torch.bfloat16)
    hmm.paged_quant_append(None, x, x, pages, pages.clone(), table, cu, kv_len)
    k, _ = hmm.paged_quant_read(pages, pages, table, cu, kv_len, 3)
    assert np.array_equal(k.double().cpu().numpy(), stored(x.double().cpu().numpy(), "int8"))
    assert (pages[:-1, :, :, 0] == 0).all()

"""paged_kv_append (norm of query and key heads, rotation, store into the paged cache)
against the formulas in float64.

Tolerance: the result is rounded once, off by at most half a step relative to its value
(finfo.eps / 2; below the smallest normal number half the smallest subnormal).  Before
that, fp32: the sum of at most 512 squares in a tree of 8 + 8 + 5 additions and its root
are off by at most 11 * 2^-24, the division, the root and two products by 4 * 2^-24, the
rotation by 3 * 2^-24 of |a| + |b|: together less than 2^-19 (|a| + |b|)."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_BOUNDS, HmmError
from heteromm_b200.paged import check_status

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def layout(new, kv, pt, hk, d, dtype, cuda, seed, spare=2):
    """A cache, a shuffled page table and the batch's vectors."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    counts = [-(-x // pt) for x in kv]
    n_pages = sum(counts) + spare
    k = torch.randn((n_pages, hk, pt, d), generator=g, device=cuda).to(dtype)
    v = torch.randn((n_pages, hk, pt, d), generator=g, device=cuda).to(dtype)
    perm = torch.randperm(n_pages, generator=g, device=cuda).to(torch.int32).cpu()
    table = torch.full((len(new), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = perm[at:at + c]
        at += c
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    return k, v, table.to(cuda), cu.to(cuda), torch.tensor(kv, dtype=torch.int32, device=cuda)


def reference(x, w, rope_rows, interleaved, eps):
    """(y, |a| + |b|) in float64; x [n, heads, D], rope_rows [n, pairs, 2] or None."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    mag = y.abs()
    if rope_rows is None:
        return y, mag
    half = rope_rows.shape[1]
    c, s = rope_rows[:, None, :, 0].double(), rope_rows[:, None, :, 1].double()
    out, mag = y.clone(), mag.clone()
    ia = torch.arange(half, device=x.device) * 2 if interleaved else torch.arange(half, device=x.device)
    ib = ia + 1 if interleaved else ia + half
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return out, mag


def close(got, ref, mag, what):
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + (1 + fi.eps) * 2.0 ** -19 * mag + fi.smallest_normal * fi.eps
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - ref).abs().max()))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,rotary,interleaved", [
    (128, 128, False), (128, 64, True), (128, 36, False), (80, 80, False), (80, 36, True),
    (80, 16, False), (64, 64, False), (8, 8, False), (8, 2, True), (256, 256, False),
    (512, 512, False), (512, 100, False), (328, 328, True), (128, 0, False)])
def test_append_formula(cuda, dtype, d, rotary, interleaved):
    new, kv, pt, hq, hk = [1, 0, 5, 19], [1, 7, 33, 20], 8, 6, 3
    dt = DT[dtype]
    k_pages, v_pages, table, cu, kv_len = layout(new, kv, pt, hk, d, dt, cuda, 11 + d)
    total = sum(new)
    g = torch.Generator(device=cuda).manual_seed(d)
    qkv = (3 * torch.randn((total + 4, hq + 2 * hk, d), generator=g, device=cuda)).to(dt)   # 4 rows of padding
    q, k, v = qkv.split([hq, hk, hk], dim=1)
    wq = (1 + 0.2 * torch.randn(d, generator=g, device=cuda)).to(dt)
    wk = (1 + 0.2 * torch.randn(d, generator=g, device=cuda)).to(dt)
    rope = hmm.rope_table(64, rotary, 500.0, cuda) if rotary else None
    out = torch.full((total + 4, hq, d), 7.0, dtype=dt, device=cuda)
    k0, v0 = k_pages.clone(), v_pages.clone()
    r = hmm.paged_kv_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope, q_weight=wq,
                            k_weight=wk, eps=1e-5, interleaved=interleaved, out=out)
    assert r is out
    assert (out[total:] == 7.0).all()          # rows that no sequence owns
    seq = np.repeat(np.arange(4), new)
    pos = np.concatenate([np.arange(x - n, x) for n, x in zip(new, kv)])
    rows = rope[torch.from_numpy(pos).to(cuda)] if rotary else None
    ref, mag = reference(q[:total], wq, rows, interleaved, 1e-5)
    close(out[:total], ref, mag, "q")
    ref, mag = reference(k[:total], wk, rows, interleaved, 1e-5)
    phys = table.cpu().numpy()[seq, pos // pt]
    got_k = k_pages[torch.from_numpy(phys).long().to(cuda), :, torch.from_numpy(pos % pt).to(cuda)]
    close(got_k, ref, mag, "k")
    got_v = v_pages[torch.from_numpy(phys).long().to(cuda), :, torch.from_numpy(pos % pt).to(cuda)]
    assert torch.equal(got_v, v[:total])
    # every other slot as it was
    mask = torch.zeros(k_pages.shape[0], pt, dtype=torch.bool, device=cuda)
    mask[torch.from_numpy(phys).long().to(cuda), torch.from_numpy(pos % pt).to(cuda)] = True
    assert torch.equal(k_pages.transpose(1, 2)[~mask], k0.transpose(1, 2)[~mask])
    assert torch.equal(v_pages.transpose(1, 2)[~mask], v0.transpose(1, 2)[~mask])


@pytest.mark.parametrize("hq,hk", [(1, 1), (0, 2), (32, 8), (7, 7), (130, 1)])
def test_append_heads_weights_positions(cuda, hq, hk):
    """No queries, many heads; fp32 weights, one of them missing; angles of given positions."""
    d, pt, new, kv = 64, 16, [3, 1], [40, 17]
    k_pages, v_pages, table, cu, kv_len = layout(new, kv, pt, hk, d, torch.bfloat16, cuda, 5)
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn((4, hq, d), generator=g, device=cuda).to(torch.bfloat16) if hq else None
    k = torch.randn((4, hk, d), generator=g, device=cuda).to(torch.bfloat16)
    v = torch.randn((4, hk, d), generator=g, device=cuda).to(torch.bfloat16)
    wk = 1 + 0.3 * torch.randn(d, generator=g, device=cuda)
    rope = hmm.rope_table(100, 32, 10000.0, cuda)
    positions = torch.tensor([99, 0, 5, 50], dtype=torch.int32, device=cuda)
    out = hmm.paged_kv_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope, k_weight=wk,
                              positions=positions)
    rows = rope[positions.long()]
    if hq:
        ref, mag = reference(q, None, rows, False, 1e-6)
        close(out, ref, mag, "q")
    else:
        assert out is None
    ref, mag = reference(k, wk, rows, False, 1e-6)
    slots = [(0, 37), (0, 38), (0, 39), (1, 16)]
    for i, (s, p) in enumerate(slots):
        close(k_pages[table[s, p // pt].item(), :, p % pt], ref[i], mag[i], "k")
        assert torch.equal(v_pages[table[s, p // pt].item(), :, p % pt], v[i])


def test_append_strided_caches_in_place_and_bits(cuda):
    """Token-major pages, K and V in one array, bf16 bits as int16, q rotated in place."""
    n_pages, pt, hk, hq, d = 9, 4, 2, 4, 128
    both = torch.zeros((n_pages, 2, pt, hk, d), dtype=torch.int16, device=cuda)
    k_pages, v_pages = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn((6, hq + 2 * hk, d), generator=g, device=cuda).to(torch.bfloat16)
    q, k, v = x.clone().view(torch.int16).split([hq, hk, hk], dim=1)
    table = torch.tensor([[8, 0, 3]], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 6], dtype=torch.int32, device=cuda)
    kv_len = torch.tensor([10], dtype=torch.int32, device=cuda)
    rope = hmm.rope_table(16, 128, 10000.0, cuda)
    r = hmm.paged_kv_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope, out=q)
    assert r is q
    ref, mag = reference(x, None, rope[4:10], False, 0.0)
    close(q.view(torch.bfloat16), ref[:, :hq], mag[:, :hq], "q")
    for i, p in enumerate(range(4, 10)):
        page = int(table[0, p // pt])
        close(both[page, 0, p % pt].view(torch.bfloat16), ref[i, hq:hq + hk], mag[i, hq:hq + hk], "k")
        assert torch.equal(both[page, 1, p % pt], v[i])


def test_append_flags(cuda):
    """A bad page, a position without an angle, a length beyond the table, a sequence
    longer than its cache: flagged, their tokens skipped, the others stored."""
    d, pt, hk = 64, 4, 1
    new, kv = [2, 1, 1, 3, 1], [6, 4, 3, 2, 99]
    k_pages, v_pages, table, cu, kv_len = layout([2, 1, 1, 3, 1], [6, 4, 3, 4, 8], pt, hk, d,
                                                 torch.float16, cuda, 3)
    kv_len = torch.tensor(kv, dtype=torch.int32, device=cuda)
    good_row = int(table[2, 0])
    table[0, 1] = k_pages.shape[0]       # tokens 0, 1 of the batch are at positions 4, 5
    table[1, 0] = -1
    k = torch.randn((8, hk, d), device=cuda).to(torch.float16)
    k0 = k_pages.clone()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    hmm.paged_kv_append(None, k, k, k_pages, v_pages, table, cu, kv_len, status=status)
    with pytest.raises(HmmError) as e:
        check_status(status)
    assert e.value.status == HMM_ERR_BOUNDS
    assert status.item() == 1 | 16
    changed = (k_pages != k0).any(-1).any(1).nonzero().cpu().tolist()
    # sequence 2's token; sequence 3 has two of its three tokens at positions 0 and 1
    assert sorted(changed) == sorted([[good_row, 2], [int(table[3, 0]), 0], [int(table[3, 0]), 1]])
    # an angle out of range, raised by the waiting form
    rope = hmm.rope_table(2, 64, device=cuda)
    with pytest.raises(HmmError) as e:
        hmm.paged_kv_append(None, k[:1], k[:1], k_pages, v_pages, table[2:3].contiguous(),
                            torch.tensor([0, 1], dtype=torch.int32, device=cuda), kv_len[2:3], rope)
    assert e.value.status == HMM_ERR_BOUNDS


def test_append_many_sequences_and_stream(cuda):
    """Every sequence of a large ragged batch finds its rows; on a stream of its own."""
    rng = np.random.RandomState(0)
    new = rng.randint(0, 4, 1500).tolist()
    kv = [n + int(x) for n, x in zip(new, rng.randint(0, 30, 1500))]
    d, pt, hk = 16, 8, 1
    k_pages, v_pages, table, cu, kv_len = layout(new, kv, pt, hk, d, torch.bfloat16, cuda, 4)
    total = sum(new)
    k = torch.randn((total, hk, d), device=cuda).to(torch.bfloat16)
    v = torch.randn((total, hk, d), device=cuda).to(torch.bfloat16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        hmm.paged_kv_append(None, k, v, k_pages, v_pages, table, cu, kv_len)
    torch.cuda.current_stream().wait_stream(st)
    seq = np.repeat(np.arange(1500), new)
    pos = np.concatenate([np.arange(x - n, x) for n, x in zip(new, kv)])
    phys = torch.from_numpy(table.cpu().numpy()[seq, pos // pt]).long().to(cuda)
    row = torch.from_numpy(pos % pt).to(cuda)
    assert torch.equal(k_pages[phys, :, row], k)
    assert torch.equal(v_pages[phys, :, row], v)

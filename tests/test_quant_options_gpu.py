"""Options of the calls over a cache in 8 bits and over shared prefixes, each against its
definition in float64: angles of given positions and norm weights in fp32 with
paged_quant_append; strides, bf16 bits and page layouts with paged_prefix_attention.  Tolerances:
test_quant_cache_gpu.py, test_prefix_attention_gpu.py."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HmmError
from test_prefix_attention_gpu import shared, with_join
from test_quant_attention_gpu import filled
from test_quant_cache_gpu import DT, decoded, layout, least_scale, places, stored
from test_serve_append_gpu import close
from test_serve_append_gpu import reference as turned
from test_serve_attention_gpu import check, reference

pytestmark = pytest.mark.gpu

NAN = float("nan")


def near(got, s, ref, mag, kind):
    """Keys that were rounded once from fp32 values off by 2^-19 of |a| + |b|."""
    e = s.astype(np.int64) - 127
    assert (e >= least_scale(ref * (1 - 2.0 ** -18), kind)).all() and (e <= least_scale(ref * (1 + 2.0 ** -18), kind)).all()
    scale = np.repeat(np.ldexp(1.0, e), 32, -1)
    half = scale / 2 if kind == "int8" else np.maximum(np.abs(ref) * 2.0 ** -4, scale * 2.0 ** -10)
    assert (np.abs(got - ref) <= half * (1 + 2.0 ** -10) + 2.0 ** -18 * mag).all()


@pytest.mark.parametrize("kind,dtype", [("e4m3", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("d,rotary,interleaved", [(128, 128, False), (64, 32, True), (96, 20, False), (256, 256, False)])
@pytest.mark.parametrize("weights", ["both", "q", "k", "none"])
def test_positions_and_fp32_weights(cuda, kind, dtype, d, rotary, interleaved, weights):
    new, kv, pt, hq, hk = [3, 0, 1, 9], [20, 4, 1, 40], 16, 4, 2
    k_pages, v_pages, table, cu, kv_len = layout(new, kv, pt, hk, d, kind, cuda, 200 + d)
    n = sum(new)
    g = torch.Generator(device=cuda).manual_seed(d)
    q, k, v = (2 * torch.randn((n, hq + 2 * hk, d), generator=g, device=cuda)).to(DT[dtype]).split([hq, hk, hk], dim=1)
    wq, wk = (1 + 0.2 * torch.randn(d, generator=g, device=cuda) for _ in range(2))          # fp32
    wq, wk = wq if weights in ("both", "q") else None, wk if weights in ("both", "k") else None
    rope = hmm.rope_table(500, rotary, 500.0, cuda)
    positions = torch.randint(0, 500, (n,), generator=g, device=cuda, dtype=torch.int32)
    positions[0], positions[1] = 499, 0
    out = hmm.paged_quant_append(q, k, v, k_pages, v_pages, table, cu, kv_len, rope, q_weight=wq, k_weight=wk, eps=1e-5,
                                 interleaved=interleaved, positions=positions)
    rows = rope[positions.long()]
    ref, mag = turned(q, wq, rows, interleaved, 1e-5)
    close(out, ref, mag, "q")
    phys, slot, _ = places(new, kv, pt, table)
    got, s = (x[phys, :, slot] for x in decoded(k_pages, kind))
    ref, mag = (x.cpu().numpy() for x in turned(k, wk, rows, interleaved, 1e-5))
    near(got, s, ref, mag, kind)
    assert np.array_equal(decoded(v_pages, kind)[0][phys, :, slot], stored(v.double().cpu().numpy(), kind))


def test_positions_out_of_bounds(cuda):
    """A token whose angle is not in the table is flagged and skipped, the others are done."""
    new, kv, pt, hk, d = [4], [10], 16, 1, 64
    k_pages, v_pages, table, cu, kv_len = layout(new, kv, pt, hk, d, "int8", cuda, 210)
    x = torch.randn((4, hk, d), device=cuda).to(torch.bfloat16)
    before = decoded(v_pages, "int8")[0]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    rope = hmm.rope_table(8, d, 500.0, cuda)
    positions = torch.tensor([0, 8, -1, 7], dtype=torch.int32, device=cuda)
    hmm.paged_quant_append(None, x, x, k_pages, v_pages, table, cu, kv_len, rope, positions=positions, status=status)
    assert status.item() == 16
    after = decoded(v_pages, "int8")[0]
    want = before.copy()
    want[table[0, 0].item(), :, [6, 9]] = stored(x.double().cpu().numpy(), "int8")[[0, 3]]
    assert np.array_equal(after, want)


GROUPS, NEW, KV = [(0, 4, 150), (5, 8, 40)], [1, 3, 40, 1, 2, 1, 5, 1], [160, 200, 230, 151, 30, 60, 45, 41]


@pytest.mark.parametrize("kind", [None, "e4m3", "int8"])
@pytest.mark.parametrize("what", ["qkv", "bits", "interleaved", "token major", "one head", "out"])
def test_layouts_of_the_prefix_call(cuda, what, kind):
    hq, hk = (2, 1) if what == "one head" else (8, 2)
    d, pt = 64, 16
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 220, GROUPS, NEW, KV, hq, hk, d, pt, torch.bfloat16)
    kp, vp = k, v
    if kind:
        kp, vp, k, v = filled(k, v, kind)
    ref = with_join(reference(q, k, v, table, NEW, KV))
    kw = {}
    if what == "qkv":                                     # heads of a wider projection
        wide = torch.full((sum(NEW), hq + 2 * hk, d + 8), NAN, dtype=torch.bfloat16, device=cuda)
        wide[:, 1:1 + hq, :d] = q
        q = wide[:, 1:1 + hq, :d]
    elif what == "bits":
        q = q.view(torch.int16)
        if not kind:
            kp, vp = kp.view(torch.int16), vp.view(torch.int16)
    elif what == "interleaved":                           # K and V pages in one array
        t = kp.dtype
        both = torch.stack([kp.view(torch.uint8), vp.view(torch.uint8)], 1).view(t)
        kp, vp = both[:, 0], both[:, 1]
    elif what == "token major" and not kind:
        kp, vp = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kp, vp))
    elif what == "token major":                           # a page and head is one block: refused
        kp, vp = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kp, vp))
        with pytest.raises(ValueError, match="one block"):
            hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl)
        return
    elif what == "one head":
        kp, vp = kp[:, 0], vp[:, 0]
    elif what == "out":
        kw["out"] = torch.full((sum(NEW), hq, d), 9.0, dtype=torch.bfloat16, device=cuda)
    out, lse = hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, return_lse=True, **kw)
    assert out.dtype == q.dtype and ("out" not in kw or out is kw["out"])
    check(out.view(torch.bfloat16), lse, ref)


@pytest.mark.parametrize("kind", [None, "int8"])
def test_status_and_lse_of_the_prefix_call_on_a_stream(cuda, kind):
    """A zero scale and a negative one, on a stream of its own, with a status word."""
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 221, GROUPS, NEW, KV, 8, 2, 128, 16, torch.float16, pad=3)
    kp, vp = k, v
    if kind:
        kp, vp, k, v = filled(k, v, kind)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    st = torch.cuda.Stream()
    for scale in (0.0, -0.11):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            out, lse = hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, scale=scale, max_new=40, return_lse=True,
                                                  status=status)
        st.synchronize()
        check(out, lse, with_join(reference(q, k, v, table, NEW, KV, scale=scale)))
    assert status.item() == 0
    with pytest.raises(ValueError, match="max_new"):
        hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, max_new=-1)
    with pytest.raises((ValueError, HmmError)):
        hmm.paged_prefix_attention(q, kp, vp, table, cu, kv_len, cg, pl, out=q)

"""The workspace of a windowed call over a cache in 8 bits: without room for keys that it would not
widen, and never written behind its end."""
import ctypes as C

import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_DTYPE_BF16, HMM_DTYPE_E4M3, HMM_ERR_OOM, HMM_OK, PagedBatch, PagedQuant
from test_quant_refusals import attend, quant
from test_serve_refusals import batch, refused

SIZES = [  # n_seq, n_tokens, hq, hk, d, max_kv, max_new
    (8, 1500, 16, 16, 64, 16000, 0), (8, 1500, 16, 16, 64, 16000, 1001), (3, 941, 64, 8, 64, 6000, 0),
    (1, 8192, 32, 8, 128, 8192, 0), (64, 64, 32, 8, 128, 16384, 1), (1, 1, 1, 1, 32, 0, 0),
]


def sizes(case, window):
    lib = hmm.load()
    return (lib.hmm_paged_quant_window_attention_workspace_size(*case, window),
            lib.hmm_paged_quant_attention_workspace_size(*case), lib.hmm_paged_attention_workspace_size(*case[:5]))


@pytest.mark.parametrize("case", SIZES)
def test_size(case):
    n_seq, n_tokens, hq, hk, d, max_kv, max_new = case
    for window in (0, 1, 100, 1024, 4000, 1 << 20, 1 << 40):
        need, most, plain = sizes(case, window)
        assert plain <= need <= most
        if window == 0 or window >= max_kv:
            assert need == most
    # products of 256 rows and 128 keys: 5 row blocks of 16 heads, 10 tiles in a window of 1,024, 125 without
    if case == SIZES[0]:
        assert sizes(case, 1024)[0] == sizes(case, 1024)[2] and sizes(case, 0)[0] > 100 << 20
    bad = hmm.load().hmm_paged_quant_window_attention_workspace_size
    assert bad(*case, -1) == 0 and bad(-1, *case[1:], 4) == 0


def test_refusal():
    c = quant(n_kv_heads=16, page_tokens=64, k_page=1 << 20, k_head=1 << 15, v_page=1 << 20, v_head=1 << 15)
    b = batch(n_seq=8, n_tokens=1500, pages_per_seq=250)
    for window, size in ((1024, sizes(SIZES[0], 1024)[0]), (0, sizes(SIZES[0], 0)[0]), (1 << 30, sizes(SIZES[0], 0)[0])):
        for n in (0, size - 1):
            refused(attend(c, b, n_heads=16, q_token=1024, window=window, nbytes=n), "workspace too small", HMM_ERR_OOM)


@pytest.mark.gpu
@pytest.mark.parametrize("new,kv,hq,hk,window,widens", [
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 2000, True),
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 300, False),
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 7000, True),
    ([1, 1, 1], [900, 300, 2900], 32, 8, 500, False),
])
def test_a_call_keeps_to_it(cuda, new, kv, hq, hk, window, widens):
    from test_quant_attention_gpu import filled
    from test_serve_attention_gpu import check, make, reference
    d, pt = 64, 16
    q, k, v, table, cu, kv_len = make(cuda, 110, new, kv, hq, hk, d, pt, torch.bfloat16, pad=20)
    kp, vp, k, v = filled(k, v, "e4m3")
    n, max_kv = q.shape[0], table.shape[1] * pt
    need, most, plain = sizes((len(new), n, hq, hk, d, max_kv, 0), window)
    assert (need > plain + (1 << 20)) == widens
    ws = torch.full((need + (1 << 20),), 171, dtype=torch.uint8, device=cuda)
    cache = PagedQuant(kp.data_ptr(), vp.data_ptr(), kp.shape[0], hk, pt, d, kp.stride(0), kp.stride(1), vp.stride(0), vp.stride(1),
                       HMM_DTYPE_E4M3)
    b = PagedBatch(table.data_ptr(), len(new), table.shape[1], cu.data_ptr(), n, kv_len.data_ptr())
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=cuda)
    r = hmm.load().hmm_paged_quant_attention(C.byref(cache), C.byref(b), HMM_DTYPE_BF16, q.data_ptr(), hq * d, d, hq, 0.125, 1,
                                             window, 3, 0, out.data_ptr(), None, status.data_ptr(), ws.data_ptr(), need,
                                             torch.cuda.current_stream().cuda_stream)
    assert r == HMM_OK and status.item() == 0
    assert (ws[need:] == 171).all()
    check(out, None, reference(q, k.contiguous(), v.contiguous(), table, new, kv, window=window, sinks=3, scale=0.125))
    again = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, window=window, sinks=3, scale=0.125)
    assert torch.equal(again[:sum(new)], out[:sum(new)])

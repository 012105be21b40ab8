"""What the serving entry points refuse before they touch the device: through the C ABI,
each case one change to a call that would be taken, and through the Python wrappers.  The
pointers are never followed."""
import ctypes as C

import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import (HMM_DTYPE_BF16, HMM_DTYPE_F32, HMM_ERR_INVALID, HMM_ERR_OOM, HMM_OK, PagedBatch,
                                PagedCache, PagedState, PageStore)

P = 0x100000


def cache(**kw):
    d = dict(k=P, v=P, n_pages=8, n_kv_heads=2, page_tokens=16, D=64, k_page=2048, k_head=1024, k_token=64,
             v_page=2048, v_head=1024, v_token=64, dtype=HMM_DTYPE_BF16)
    d.update(kw)
    return PagedCache(*[d[n] for n, _ in PagedCache._fields_])


def batch(**kw):
    d = dict(page_table=P, n_seq=2, pages_per_seq=4, cu_new=P, n_tokens=5, kv_len=P)
    d.update(kw)
    return PagedBatch(*[d[n] for n, _ in PagedBatch._fields_])


def store(**kw):
    d = dict(k=P, v=P, n_pages=8, page_bytes=4096, n_layers=2, k_page=4096, k_layer=32768, v_page=4096,
             v_layer=32768)
    d.update(kw)
    return PageStore(*[d[n] for n, _ in PageStore._fields_])


def state(**kw):
    d = dict(table_in=P, refs_in=P, kv_len_in=P, table_out=P, refs_out=P, kv_len_out=P, n_seq=2, pages_per_seq=4,
             n_pages=8)
    d.update(kw)
    return PagedState(*[d[n] for n, _ in PagedState._fields_])


def refused(got, text, code=HMM_ERR_INVALID):
    assert got == code and text in hmm.last_error(), (got, hmm.last_error())


BAD_CACHE = [
    (dict(dtype=HMM_DTYPE_F32), "dtype"),
    (dict(dtype=9), "dtype"),
    (dict(D=0), "D must"),
    (dict(D=68), "D must"),
    (dict(D=520), "D must"),
    (dict(n_kv_heads=0), "n_kv_heads"),
    (dict(n_kv_heads=65536), "n_kv_heads"),
    (dict(page_tokens=0), "page_tokens"),
    (dict(page_tokens=1 << 31), "page_tokens"),
    (dict(page_tokens=1 << 30), "2^31"),
    (dict(n_pages=-1), "n_pages"),
    (dict(n_pages=1 << 31), "n_pages"),
    (dict(k_page=2044), "strides"),
    (dict(v_head=-8), "strides"),
    (dict(v_token=65), "strides"),
    (dict(k=P + 8), "aligned"),
    (dict(v=P + 2), "aligned"),
    (dict(k=None), "null page array"),
]
BAD_BATCH = [
    (dict(n_seq=-1), "n_seq"),
    (dict(n_seq=65536), "n_seq"),
    (dict(pages_per_seq=-1), "pages_per_seq"),
    (dict(n_tokens=-1), "n_tokens"),
    (dict(n_tokens=(1 << 30) + 1), "n_tokens"),
    (dict(pages_per_seq=1 << 28), "2^31"),
    (dict(cu_new=None), "null cu_new"),
    (dict(kv_len=None), "kv_len"),
    (dict(page_table=None), "null page table"),
]


def attend(c=None, b=None, q=P, q_token=256, q_head=64, n_heads=4, scale=0.125, causal=1, window=0, sinks=0, max_new=0,
           out=P, status=P, ws=P, nbytes=1 << 40):
    return hmm.load().hmm_paged_attention(C.byref(c or cache()), C.byref(b or batch()), q, q_token, q_head, n_heads,
                                          scale, causal, window, sinks, max_new, out, None, status, ws, nbytes, None)


def append(c=None, b=None, q=P, q_token=256, n_heads=4, k=P, k_token=128, v=P, weights=(None, None), weight_dtype=-1,
           eps=1e-6, rope=P, n_pos=64, rotary=64, q_out=P, status=P):
    return hmm.load().hmm_paged_kv_append(C.byref(c or cache()), C.byref(b or batch()), q, q_token, 64, n_heads, k,
                                          k_token, 64, v, 128, 64, *weights, weight_dtype, eps, rope, n_pos, rotary,
                                          0, None, q_out, 256, 64, status, None)


@pytest.mark.parametrize("change,text", BAD_CACHE)
def test_bad_cache(change, text):
    refused(attend(cache(**change)), text)
    refused(append(cache(**change)), text)


@pytest.mark.parametrize("change,text", BAD_BATCH)
def test_bad_batch(change, text):
    refused(attend(b=batch(**change)), text)
    refused(append(b=batch(**change)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(n_heads=0), "n_heads"), (dict(n_heads=3), "n_heads"), (dict(n_heads=65538), "n_heads"),
    (dict(status=None), "device_status"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks"),
    (dict(causal=0, window=4), "causal"), (dict(causal=0, sinks=4), "causal"), (dict(max_new=-1), "max_new"),
    (dict(q_token=100), "q strides"), (dict(q_head=-64), "q strides"), (dict(q=None), "null q"),
    (dict(out=None), "null q or out"), (dict(q=P + 2), "aligned"), (dict(out=P + 8), "aligned"),
    (dict(ws=P + 8), "aligned"), (dict(c=cache(D=264)), "D must"), (dict(c=cache(n_pages=0)), "no pages"),
    (dict(c=cache(k_token=0)), "strides"), (dict(c=cache(v_page=0)), "strides"), (dict(c=cache(k_head=0)), "strides"),
    (dict(c=cache(k_page=1 << 39)), "strides"),
    (dict(c=cache(page_tokens=1 << 20), b=batch(pages_per_seq=(1 << 11) - 1), n_heads=65534,
          q=None), "null q"),
    (dict(c=cache(page_tokens=(1 << 31) - 512), b=batch(pages_per_seq=1)), "2^31 - 1024"),
    (dict(c=cache(n_kv_heads=1), b=batch(n_tokens=1 << 30), n_heads=4), "2^31"),
])
def test_bad_attention(kw, text):
    refused(attend(**kw), text)


def test_out_over_q():
    """Default calls here have out = q, which is refused last; rows of out would be read."""
    refused(attend(), "overlaps")
    span = (4 * 256 + 3 * 64 + 64) * 2                 # bytes of q
    refused(attend(out=P + span - 16), "overlaps")
    refused(attend(out=P - 5 * 4 * 64 * 2 + 16), "overlaps")


def test_attention_workspace():
    lib = hmm.load()
    need = lib.hmm_paged_attention_workspace_size(2, 5, 4, 2, 64)
    assert need > 0
    refused(attend(nbytes=need - 1), "workspace", HMM_ERR_OOM)
    refused(attend(ws=None), "workspace", HMM_ERR_OOM)
    for sizes in ((-1, 5, 4, 2, 64), (2, -1, 4, 2, 64), (2, 5, 0, 2, 64), (2, 5, 4, 0, 64), (2, 5, 4, 2, 0),
                  (2, 5, 4, 2, 264)):
        assert lib.hmm_paged_attention_workspace_size(*sizes) == 0
    # more of anything never needs less
    for d in (64, 128, 256):
        a = lib.hmm_paged_attention_workspace_size(4, 10000, 8, 2, d)
        assert a <= lib.hmm_paged_attention_workspace_size(400, 10000, 8, 2, d)


@pytest.mark.parametrize("kw,text", [
    (dict(n_heads=-1), "n_heads"), (dict(n_heads=65536), "n_heads"), (dict(status=None), "device_status"),
    (dict(rotary=0), "rotary"), (dict(rotary=63), "rotary"), (dict(rotary=66), "rotary"), (dict(n_pos=-1), "n_pos"),
    (dict(weights=(P, None), weight_dtype=1), "weight"), (dict(eps=-1.0), "eps"),
    (dict(b=batch(pages_per_seq=0)), "no pages"), (dict(k=None), "null q, k"), (dict(v=None), "null q, k"),
    (dict(q=None), "null q, k"), (dict(q_out=None), "null q, k"), (dict(q=P + 4), "aligned"),
    (dict(k_token=60), "strides"), (dict(q_token=-8), "strides"),
])
def test_bad_append(kw, text):
    refused(append(**kw), text)


def test_nothing_to_do_is_taken():
    """No sequences or tokens: no launch, and null arrays are fine."""
    none = batch(n_seq=0, page_table=None, cu_new=None, kv_len=None)
    assert attend(b=none) == HMM_OK and append(b=none) == HMM_OK
    none = batch(n_tokens=0)
    assert attend(b=none, q=None, out=None) == HMM_OK and append(b=none) == HMM_OK


BAD_STORE = [
    (dict(n_pages=-1), "n_pages"), (dict(n_layers=0), "n_layers"), (dict(n_layers=32768), "n_layers"),
    (dict(page_bytes=8), "page_bytes"), (dict(page_bytes=4100), "page_bytes"), (dict(k=None), "null page array"),
    (dict(v=P + 8), "aligned"), (dict(k_page=4104), "strides"), (dict(v_layer=-16), "strides"),
    (dict(k_page=4080), ""), (dict(v_page=0), ""),
]


@pytest.mark.parametrize("change,text", BAD_STORE)
def test_bad_store(change, text):
    lib = hmm.load()
    s = store(**change)
    refused(lib.hmm_paged_copy_pages(C.byref(s), P, P, 3, P, P, 4, None), text)
    if "n_pages" not in change:
        refused(lib.hmm_paged_fork(C.byref(state()), C.byref(s), 16, P, P, 1, P, P, 1 << 30, None), text)
        refused(lib.hmm_paged_compact(C.byref(state()), C.byref(s), P, P, P, 1 << 30, None), text)


BAD_STATE = [
    (dict(n_seq=-1), "n_seq"), (dict(n_seq=65536), "n_seq"), (dict(pages_per_seq=-1), "pages_per_seq"),
    (dict(n_pages=-1), "n_pages"), (dict(table_in=None), "page table"), (dict(table_out=None), "page table"),
    (dict(refs_in=None), "refs"), (dict(refs_out=None), "refs"),
]


@pytest.mark.parametrize("change,text", BAD_STATE)
def test_bad_state(change, text):
    lib = hmm.load()
    st, big = state(**change), 1 << 40
    refused(lib.hmm_paged_free(C.byref(st), P, 1, P, P, big, None), text)
    refused(lib.hmm_paged_grow(C.byref(st), 16, P, P, P, big, None), text)
    refused(lib.hmm_paged_fork(C.byref(st), C.byref(store()), 16, P, P, 1, P, P, big, None), text)
    refused(lib.hmm_paged_compact(C.byref(st), C.byref(store()), P, P, P, big, None), text)


def test_bad_page_calls():
    lib = hmm.load()
    st, sr, big = state(), store(), 1 << 30
    refused(lib.hmm_paged_copy_pages(C.byref(sr), P, P, -1, P, P, 4, None), "n must")
    refused(lib.hmm_paged_copy_pages(C.byref(sr), P, P, 1, None, P, 4, None), "device_status")
    refused(lib.hmm_paged_copy_pages(C.byref(sr), None, P, 1, P, P, 4, None), "null src")
    refused(lib.hmm_paged_copy_pages(C.byref(sr), P, P, 1, P, P, 3, None), "workspace", HMM_ERR_OOM)
    refused(lib.hmm_paged_free(C.byref(st), None, 1, P, P, big, None), "null seqs")
    refused(lib.hmm_paged_free(C.byref(st), P, -1, P, P, big, None), "n must")
    need = lib.hmm_paged_state_workspace_size(2, 8)
    refused(lib.hmm_paged_free(C.byref(st), P, 1, P, P, need - 1, None), "workspace", HMM_ERR_OOM)
    refused(lib.hmm_paged_grow(C.byref(st), 0, P, P, P, big, None), "page_tokens")
    for pt in (1 << 30, 1 << 61, 1 << 62):
        refused(lib.hmm_paged_grow(C.byref(st), pt, P, P, P, big, None), "page_tokens")
        refused(lib.hmm_paged_fork(C.byref(st), C.byref(sr), pt, P, P, 1, P, P, big, None), "page_tokens")
    refused(lib.hmm_paged_grow(C.byref(state(pages_per_seq=0)), 1 << 40, P, P, P, big, None), "page_tokens")
    refused(lib.hmm_paged_grow(C.byref(st), 16, None, P, P, big, None), "null n_new")
    refused(lib.hmm_paged_grow(C.byref(state(kv_len_in=None)), 16, P, P, P, big, None), "kv_len")
    refused(lib.hmm_paged_fork(C.byref(st), C.byref(store(n_pages=9)), 16, P, P, 1, P, P, big, None), "the store has")
    refused(lib.hmm_paged_fork(C.byref(st), C.byref(sr), 16, P, None, 1, P, P, big, None), "null src")
    refused(lib.hmm_paged_compact(C.byref(st), C.byref(sr), None, P, P, big, None), "null out_live")
    refused(lib.hmm_paged_compact(C.byref(st), C.byref(store(n_pages=9)), P, P, P, big, None), "the store has")


def test_wrappers_refuse_host_tensors():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    t, cu, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_attention(q, k, k, t, cu, n)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_attention(q=q, k_pages=k, v_pages=k, page_table=t, cu_new=cu, kv_len=n)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_kv_append(q, q, q, k, k, t, cu, n)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_copy_pages(k, k, n, n)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_free(t, n, n, n)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_grow(t, n, n, n, 16)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_fork(t, n, n, n, n, k, k)
    with pytest.raises(ValueError, match="CUDA"):
        hmm.paged_compact(t, n, k, k)
    for dim in (0, 3, -2):
        with pytest.raises(ValueError, match="rotary_dim"):
            hmm.rope_table(4, dim, device="cpu")


def test_rope_table():
    t = hmm.rope_table(70000, 6, theta=1e4, device="cpu")
    assert t.shape == (70000, 3, 2) and t.dtype == torch.float32
    a = torch.tensor(69999.0, dtype=torch.float64) * 1e4 ** (-torch.arange(3, dtype=torch.float64) / 3)
    assert torch.equal(t[69999, :, 0], a.cos().float()) and torch.equal(t[69999, :, 1], a.sin().float())
    assert hmm.rope_table(0, 2, device="cpu").shape == (0, 1, 2)

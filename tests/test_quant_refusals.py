"""What the calls of a cache held in 8 bits refuse before they touch the device: through the C
ABI, each case one change to a call that would be taken, and through the Python wrappers.  The
pointers are never followed."""
import ctypes as C

import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import (HMM_DTYPE_BF16, HMM_DTYPE_E4M3, HMM_DTYPE_F16, HMM_DTYPE_F32, HMM_DTYPE_I8, HMM_ERR_OOM,
                                HMM_OK,
                                PagedQuant)
from test_serve_refusals import BAD_BATCH, BAD_CACHE, P, batch, cache, refused

FAR = 1 << 30


def quant(**kw):
    """Pages of 16 tokens, 2 heads of 64: 1,056 bytes a page and head."""
    d = dict(k=P, v=P, n_pages=8, n_kv_heads=2, page_tokens=16, D=64, k_page=2112, k_head=1056, v_page=2112, v_head=1056,
             codes=HMM_DTYPE_E4M3)
    d.update(kw)
    return PagedQuant(*[d[n] for n, _ in PagedQuant._fields_])


BAD_QUANT = [
    (dict(codes=HMM_DTYPE_BF16), "codes must"), (dict(codes=5), "codes must"),
    (dict(D=0), "D must"), (dict(D=48), "D must"), (dict(D=288), "D must"), (dict(D=16), "D must"),
    (dict(n_kv_heads=0), "n_kv_heads"), (dict(n_kv_heads=65536), "n_kv_heads"),
    (dict(page_tokens=0), "page_tokens"), (dict(page_tokens=1 << 30), "2^31"),
    (dict(page_tokens=4), "multiple of 16"), (dict(page_tokens=12), "multiple of 16"), (dict(page_tokens=8, D=96), "multiple of 16"),
    (dict(n_pages=-1), "n_pages"), (dict(n_pages=1 << 31), "n_pages"),
    (dict(k_page=2120), "strides"), (dict(v_head=-16), "strides"), (dict(v_page=1 << 40), "strides"),
    (dict(k_head=1040), "takes 1056 bytes"), (dict(v_page=1024), "takes 1056 bytes"), (dict(k_page=0), "takes 1056 bytes"),
    (dict(k=P + 8), "aligned"), (dict(v=P + 1), "aligned"), (dict(k=None), "null page array"),
]


def append(c=None, b=None, dtype=HMM_DTYPE_BF16, q=P, q_token=256, n_heads=4, k=P, k_token=128, v=P, weights=(None, None),
           weight_dtype=-1, eps=1e-6, rope=P, n_pos=64, rotary=64, q_out=P, status=P):
    return hmm.load().hmm_paged_quant_append(C.byref(c or quant()), C.byref(b or batch()), dtype, q, q_token, 64, n_heads,
                                             k, k_token, 64, v, 128, 64, *weights, weight_dtype, eps, rope, n_pos, rotary,
                                             0, None, q_out, 256, 64, status, None)


def read(c=None, b=None, dtype=HMM_DTYPE_BF16, k=P + FAR, v=P + 2 * FAR, status=P):
    return hmm.load().hmm_paged_quant_read(C.byref(c or quant()), C.byref(b or batch()), dtype, k, v, status, None)


def attend(c=None, b=None, dtype=HMM_DTYPE_BF16, q=P, q_token=256, q_head=64, n_heads=4, scale=0.125, causal=1, window=0,
           sinks=0, max_new=0, out=P + FAR, status=P, ws=P, nbytes=1 << 40):
    return hmm.load().hmm_paged_quant_attention(C.byref(c or quant()), C.byref(b or batch()), dtype, q, q_token, q_head,
                                                n_heads, scale, causal, window, sinks, max_new, out, None, status, ws,
                                                nbytes, None)


def shared(c=None, b=None, cu_group=P, prefix=P, n_groups=2, q=P, q_token=256, q_head=64, n_heads=4, scale=0.125,
           out=P + FAR, status=P, ws=P, nbytes=1 << 40):
    return hmm.load().hmm_paged_prefix_attention(C.byref(c or cache()), C.byref(b or batch()), cu_group, prefix, n_groups, q,
                                                 q_token, q_head, n_heads, scale, out, None, status, ws, nbytes, None)


def shared_quant(c=None, b=None, dtype=HMM_DTYPE_BF16, cu_group=P, prefix=P, n_groups=2, q=P, q_token=256, q_head=64,
                 n_heads=4, scale=0.125, out=P + FAR, status=P, ws=P, nbytes=1 << 40):
    return hmm.load().hmm_paged_quant_prefix_attention(C.byref(c or quant()), C.byref(b or batch()), dtype, cu_group, prefix,
                                                       n_groups, q, q_token, q_head, n_heads, scale, out, None, status, ws,
                                                       nbytes, None)


@pytest.mark.parametrize("change,text", BAD_QUANT)
def test_bad_cache(change, text):
    for call in (append, read, attend, shared_quant):
        refused(call(quant(**change)), text)


@pytest.mark.parametrize("change,text", BAD_CACHE)
def test_bad_cache_of_16_bits(change, text):
    refused(shared(cache(**change)), text)


@pytest.mark.parametrize("change,text", BAD_BATCH)
def test_bad_batch(change, text):
    for call in (append, read, attend, shared, shared_quant):
        refused(call(b=batch(**change)), text)


BAD_ATTENTION = [
    (dict(n_heads=0), "n_heads"), (dict(n_heads=3), "n_heads"), (dict(n_heads=65538), "n_heads"),
    (dict(status=None), "device_status"), (dict(q_token=100), "q strides"), (dict(q_head=-64), "q strides"),
    (dict(q=None), "null q"), (dict(out=None), "null q or out"), (dict(q=P + 2), "aligned"), (dict(out=P + FAR + 8), "aligned"),
    (dict(ws=P + 8), "aligned"), (dict(out=P), "out overlaps q"),
]


@pytest.mark.parametrize("kw,text", BAD_ATTENTION)
def test_bad_attention(kw, text):
    for call in (attend, shared, shared_quant):
        refused(call(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=HMM_DTYPE_F32), "dtype must"), (dict(dtype=HMM_DTYPE_E4M3), "dtype must"), (dict(window=-1), "window"),
    (dict(sinks=-1), "sinks"), (dict(causal=0, window=4), "causal"), (dict(causal=0, sinks=4), "causal"), (dict(max_new=-1), "max_new"),
    (dict(c=quant(n_pages=0)), "no pages"), (dict(c=quant(page_tokens=(1 << 31) - 512, k_page=1 << 39, k_head=1 << 38, v_page=1 << 39,
                                                          v_head=1 << 38), b=batch(pages_per_seq=1)), "2^31 - 1024"),
    (dict(c=quant(n_kv_heads=1), b=batch(n_tokens=1 << 30), n_heads=4), "2^31"),
])
def test_bad_quant_attention(kw, text):
    refused(attend(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(n_groups=-1), "n_groups"), (dict(n_groups=3), "n_groups"), (dict(cu_group=None), "null cu_group"),
    (dict(prefix=None), "null cu_group"),
])
def test_bad_groups(kw, text):
    refused(shared(**kw), text)
    refused(shared_quant(**kw), text)


def test_workspaces():
    lib = hmm.load()
    for n_seq, n_tokens, heads, hk, d, max_new in ((2, 5, 4, 2, 64, 0), (64, 64, 32, 8, 128, 1), (64, 200, 32, 8, 128, 0),
                                                   (3, 99000, 7, 1, 256, 0), (1, 1, 1, 1, 32, 0), (3, 99000, 7, 1, 128, 16)):
        c = quant(n_kv_heads=hk, D=d, page_tokens=64, k_page=1 << 20, k_head=1 << 15, v_page=1 << 20, v_head=1 << 15)
        b, kw = batch(n_seq=n_seq, n_tokens=n_tokens), dict(n_heads=heads, q_token=heads * d, q_head=d)
        plain = lib.hmm_paged_attention_workspace_size(n_seq, n_tokens, heads, hk, d)
        need = lib.hmm_paged_quant_attention_workspace_size(n_seq, n_tokens, heads, hk, d, 4 * 64, max_new)
        assert plain > 0 and need >= plain
        wide = n_tokens * heads // hk // 256 * hk * 2 >= 4096 and max_new == 0      # keys may be widened into the workspace
        assert wide == (need > plain + 4 * 256 * hk * d)
        for n in (0, need - 1):
            refused(attend(c, b, max_new=max_new, nbytes=n, **kw), "workspace too small", HMM_ERR_OOM)
        for groups in (0, n_seq):
            more = lib.hmm_paged_prefix_attention_workspace_size(n_seq, n_tokens, groups, heads, hk, d)
            assert more >= plain + 8 * n_tokens * heads * (d + 1)
            refused(shared(cache(n_kv_heads=hk, D=d), b, n_groups=groups, nbytes=more - 1, **kw), "workspace too small", HMM_ERR_OOM)
            more = lib.hmm_paged_quant_prefix_attention_workspace_size(n_seq, n_tokens, groups, heads, hk, d, 4 * 64)
            refused(shared_quant(c, b, n_groups=groups, nbytes=more - 1, **kw), "workspace too small", HMM_ERR_OOM)
    assert lib.hmm_paged_quant_attention_workspace_size(1, 1, 1, 1, 257, 64, 0) == 0
    assert lib.hmm_paged_quant_attention_workspace_size(1, 1, 1, 1, 64, -1, 0) == 0
    assert lib.hmm_paged_prefix_attention_workspace_size(1, 1, -1, 1, 1, 64) == 0
    assert lib.hmm_paged_quant_prefix_attention_workspace_size(1, 1, -1, 1, 1, 64, 64) == 0
    # a long table takes no more than the limit
    assert lib.hmm_paged_quant_attention_workspace_size(64, 65536, 32, 8, 128, 1 << 20, 0) < 3 << 30


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=HMM_DTYPE_F32), "dtype must"), (dict(dtype=HMM_DTYPE_I8), "dtype must"),
    (dict(n_heads=-1), "n_heads"), (dict(status=None), "device_status"), (dict(rotary=66), "rotary_dim"),
    (dict(rotary=31), "rotary_dim"), (dict(n_pos=-1), "n_pos"), (dict(weights=(P, None), weight_dtype=HMM_DTYPE_F16), "norm weights"),
    (dict(eps=-1.0), "eps"), (dict(k=None), "null q, k, v"), (dict(q=None), "null q, k, v"), (dict(v=P + 8), "aligned"),
    (dict(q_token=100), "row strides"), (dict(b=batch(pages_per_seq=0)), "no pages"),
    (dict(q_out=P + 128, k=P + FAR, v=P + FAR), "overlap"), (dict(q=P + FAR, v=P + FAR), "overlaps k or v"),
])
def test_bad_append(kw, text):
    refused(append(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=HMM_DTYPE_E4M3), "dtype must"), (dict(dtype=7), "dtype must"), (dict(status=None), "device_status"),
    (dict(k=None), "null k_out"), (dict(v=None), "null k_out"), (dict(k=P + FAR + 8), "aligned"),
    (dict(v=P + FAR + 1264), "k_out and v_out overlap"), (dict(v=P + FAR), "k_out and v_out overlap"),
    (dict(k=P + 16880), "overlaps the pages"), (dict(v=P - 1264), "overlaps the pages"), (dict(b=batch(pages_per_seq=0)), "no pages"),
])
def test_bad_read(kw, text):
    refused(read(**kw), text)


def test_nothing_to_do():
    for b in (batch(n_seq=0), batch(n_tokens=0)):
        assert append(b=b) == HMM_OK and read(b=b) == HMM_OK and attend(b=b) == HMM_OK
        assert shared(b=b, n_groups=0) == HMM_OK and shared_quant(b=b, n_groups=0) == HMM_OK


def test_wrappers_refuse():
    x = torch.zeros(4, 2, 16, 66, dtype=torch.int8)
    with pytest.raises(ValueError, match="k_pages must be a CUDA tensor"):
        hmm.paged_quant_read(x, x, x, x, x, 4)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        hmm.paged_quant_append(x, x, x, x, x, x, x, x)
    with pytest.raises(ValueError, match="q must be a CUDA tensor"):
        hmm.paged_quant_attention(x, x, x, x, x, x)
    with pytest.raises(ValueError, match="q must be a CUDA tensor"):
        hmm.paged_prefix_attention(x, x, x, x, x, x, x, x)
    for kw, error in ((dict(dtype=torch.uint8), TypeError), (dict(D=80), ValueError), (dict(D=288), ValueError),
                      (dict(page_tokens=4), ValueError), (dict(page_tokens=0), ValueError)):
        with pytest.raises(error):
            hmm.quant_pages(**{"n_pages": 1, "n_kv_heads": 1, "page_tokens": 16, "D": 64, "device": "cpu", **kw})
    pages = hmm.quant_pages(3, 2, 8, 64, torch.int8, "cpu")
    assert tuple(pages.shape) == (3, 2, 8, 66) and pages.dtype == torch.int8 and not pages.any()

"""Arguments of the serving entry points that overlap: refused on the host, before anything
is launched.  The pointers are never followed."""
import ctypes as C

import pytest

import heteromm_b200 as hmm
from test_serve_refusals import P, batch, cache, refused

FAR = 1 << 30


def append(out, out_token=256, out_head=64, q=P, q_token=256, q_head=64, k=P + FAR, k_token=128, v=P + 2 * FAR, v_token=128,
           n_heads=4, **b):
    """5 tokens of 4 heads of 64 values (128 bytes a row), 2 KV heads."""
    return hmm.load().hmm_paged_kv_append(C.byref(cache()), C.byref(batch(**b)), q, q_token, q_head, n_heads, k, k_token, 64,
                                          v, v_token, 64, None, None, -1, 1e-6, None, 0, 0, 0, None, out, out_token, out_head,
                                          P, None)


@pytest.mark.parametrize("kw", [
    dict(out=P + 128),                                   # a head further
    dict(out=P - 128),
    dict(out=P + 512),                                   # a token further
    dict(out=P + 16),                                    # within a row
    dict(out=P + 4 * 512 + 3 * 128 + 112),               # its last bytes
    dict(out=P, out_token=512),                          # its first row alone, other strides
    dict(out=P, out_head=128),
    dict(out=P, q_token=0),                              # one query for all tokens
    dict(out=P, out_token=512, q_token=512, n_heads=3, q_head=128, out_head=64),
])
def test_out_over_q(kw):
    refused(append(**kw), "overlap")


@pytest.mark.parametrize("kw", [
    dict(out=P + FAR), dict(out=P + 2 * FAR), dict(out=P + FAR - 512), dict(out=P + 2 * FAR + 1152),
    # q, k and v of one projection [5][8 heads][64]: out over some of it that is not q
    dict(q=P, q_token=512, k=P + 512, k_token=512, v=P + 768, v_token=512, out=P + 512, out_token=512),
    dict(q=P, q_token=512, k=P + 512, k_token=512, v=P + 768, v_token=512, out=P + 256, out_token=512),
    dict(q=P, q_token=512, k=P + 512, k_token=512, v=P + 768, v_token=512, out=P + 768 + 1024, out_token=512),
    # in place, but k is q's last head
    dict(q=P, q_token=512, k=P + 384, k_token=512, v=P + 768, v_token=512, out=P, out_token=512),
])
def test_out_over_keys_or_values(kw):
    refused(append(**kw), "overlap")


@pytest.mark.parametrize("kw", [
    dict(out_token=0), dict(out_head=0), dict(out_token=64), dict(out_token=192), dict(out_head=32),
    dict(out_token=256, out_head=128), dict(out_token=64, out_head=256),
])
def test_out_over_itself(kw):
    refused(append(out=P + 3 * FAR, **kw), "overlap")

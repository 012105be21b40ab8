"""Arguments of the serving entry points that overlap: refused on the host, before anything
is launched.  The pointers are never followed."""
import ctypes as C

import pytest

import heteromm_b200 as hmm
from test_serve_refusals import P, batch, cache, refused, state, store

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


T, R, L, V = P, P + FAR, P + 2 * FAR, P + 3 * FAR        # table, references, lengths, vectors
NEW = 8 * FAR                                            # the new state: apart


def apart(**kw):
    d = dict(table_in=T, refs_in=R, kv_len_in=L, table_out=T + NEW, refs_out=R + NEW, kv_len_out=L + NEW)
    d.update(kw)
    return state(**d)


STATES = [   # [2][4] entries, 8 references, 2 lengths
    dict(table_out=T + 16), dict(table_out=T - 28), dict(refs_out=R + 4), dict(refs_out=R - 28), dict(table_out=R),
    dict(table_out=R + 28), dict(refs_out=T), dict(table_out=R + NEW - 4), dict(refs_out=T + NEW),
    dict(table_out=T, refs_out=T + 28),
]
LENGTHS = [
    dict(kv_len_out=L + 4), dict(kv_len_out=L - 4), dict(kv_len_out=T), dict(kv_len_out=R + 28), dict(table_out=L),
    dict(refs_out=L + 4), dict(kv_len_out=T + NEW + 28), dict(kv_len_out=R + NEW),
]
VECTORS = [  # three numbers at V
    dict(table_out=V - 28), dict(table_out=V + 8), dict(refs_out=V), dict(kv_len_out=V + 8), dict(kv_len_out=V - 4),
    dict(table_out=V, table_in=V),
]
BIG = 1 << 30


@pytest.mark.parametrize("change", STATES + LENGTHS + VECTORS)
def test_states_that_overlap(change):
    lib, st = hmm.load(), apart(**change)
    refused(lib.hmm_paged_free(C.byref(st), V, 3, P, P, BIG, None), "overlap")
    refused(lib.hmm_paged_fork(C.byref(st), C.byref(store()), 16, V, V, 3, P, P, BIG, None), "overlap")
    if change not in (dict(table_out=V + 8), dict(kv_len_out=V + 8)):      # (two numbers here)
        refused(lib.hmm_paged_grow(C.byref(st), 16, V, P, P, BIG, None), "overlap")
    if change in STATES:
        refused(lib.hmm_paged_compact(C.byref(st), C.byref(store()), V + FAR, P, P, BIG, None), "overlap")


def test_one_vector_that_overlaps():
    lib, st = hmm.load(), apart()
    for out in (st.table_out, st.refs_out, st.kv_len_out):
        refused(lib.hmm_paged_fork(C.byref(st), C.byref(store()), 16, V, out, 3, P, P, BIG, None), "overlap")
        refused(lib.hmm_paged_fork(C.byref(st), C.byref(store()), 16, out, V, 3, P, P, BIG, None), "overlap")
        refused(lib.hmm_paged_grow(C.byref(st), 16, out, P, P, BIG, None), "overlap")
    for live in (st.table_out, st.refs_out + 28, T, R):
        refused(lib.hmm_paged_compact(C.byref(st), C.byref(store()), live, P, P, BIG, None), "overlap")
    # lengths that double: only in place
    refused(lib.hmm_paged_grow(C.byref(apart(kv_len_out=L + NEW)), 16, L + NEW, P, P, BIG, None), "overlap")
    refused(lib.hmm_paged_grow(C.byref(apart(kv_len_out=L)), 16, L + 4, P, P, BIG, None), "overlap")

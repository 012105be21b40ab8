"""A cache of several heads filled by paged_kv_append is, head by head, the single-head cache
of the block summaries and the block-sparse decode: page p of head h is page
p * n_kv_heads + h."""
import numpy as np
import pytest
import torch

import gen
import heteromm_b200 as hmm
from oracle import oracle as O
from test_paged_gpu import ATOL, RTOL, decode_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seq,L,hk,d,pt,bt,top", [(3, 1000, 4, 64, 16, 64, 6), (2, 2048, 2, 128, 16, 64, 32),
                                                    (2, 130, 3, 128, 8, 64, 3)])
def test_summaries_and_sparse_decode_of_a_served_cache(cuda, n_seq, L, hk, d, pt, bt, top):
    pps = -(-L // pt)
    n_pages = n_seq * pps + 3
    bits = lambda seed, shape: gen.bf16_bits(gen.normal_f32(seed, shape))      # noqa: E731
    keys, vals, q = bits(90, (n_seq, L, hk, d)), bits(91, (n_seq, L, hk, d)), bits(92, (n_seq, hk, d))
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).to(cuda)      # noqa: E731
    perm = np.random.RandomState(4).permutation(n_pages)[:n_seq * pps].astype(np.int32)
    table = torch.from_numpy(perm.reshape(n_seq, pps)).to(cuda)
    k_pages = torch.zeros((n_pages, hk, pt, d), dtype=torch.int16, device=cuda)
    v_pages = torch.zeros_like(k_pages)
    cu = torch.arange(n_seq + 1, dtype=torch.int32, device=cuda) * L
    kv_len = torch.full((n_seq,), L, dtype=torch.int32, device=cuda)
    hmm.paged_kv_append(None, dev(keys).reshape(-1, hk, d), dev(vals).reshape(-1, hk, d), k_pages, v_pages, table, cu, kv_len)
    # head by head: [n_seq * hk] sequences of one head
    one_k, one_v = k_pages.view(-1, pt, d), v_pages.view(-1, pt, d)
    heads = torch.arange(hk, dtype=torch.int32, device=cuda)[None, :, None]
    one_table = (table[:, None, :] * hk + heads).reshape(n_seq * hk, pps).contiguous()
    summ = hmm.paged_kv_summary_bf16(one_k, one_table, L, bt)
    blocks, out = hmm.block_sparse_decode_bf16(dev(q).reshape(-1, d), summ, one_k, one_v, one_table, L, bt, top)
    nb = -(-L // bt)
    for s in range(n_seq):
        for h in range(hk):
            i = s * hk + h
            ref = O.block_mean_f32(gen.bf16_to_f32(keys[s, :, h]), bt)
            assert np.array_equal(summ[i].cpu().numpy().view(np.uint32), ref.view(np.uint32))
            rb, ro = decode_oracle(np.ascontiguousarray(keys[s, :, h]), np.ascontiguousarray(vals[s, :, h]), q[s, h], bt, top)
            assert np.array_equal(blocks[i, :min(top, nb)].cpu().numpy(), rb)
            np.testing.assert_allclose(out[i].cpu().numpy(), ro, rtol=RTOL, atol=ATOL)
    if top >= nb:   # every block selected: attention of the newest token, but for its own rounding to bf16
        dense = hmm.paged_attention(dev(q), k_pages, v_pages, table, torch.arange(n_seq + 1, dtype=torch.int32, device=cuda),
                                    kv_len)
        got, want = dense.view(torch.bfloat16).double().reshape(-1, d), out.double()
        # weights and results rounded by half a step (2^-8 of the largest |v| < 6 and of the value), the scale as the decode's
        assert ((got - want).abs() <= 2.0 ** -8 * (want.abs() + 6.0) + 2.0 ** -16).all()

"""paged_quant_attention where one key outweighs the others by many orders of magnitude and holds
zeros in some columns, which are then the others' alone.

The rows kernel rounds weights to fp16, held so that a row's largest is 2^14: one is off by
2^-11 of itself or by half of fp16's smallest step, 2^-25, whichever is more, that is by 2^-39 of the
largest, whose share is at most 1.  So beside the tolerance of test_serve_attention_gpu.py a column is off by
at most n 2^-39 max |v| for n keys, whatever the queries' type."""
import pytest
import torch

import heteromm_b200 as hmm
from test_quant_attention_gpu import filled
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dtype", [("int8", "bf16"), ("e4m3", "bf16"), ("int8", "fp16")])
@pytest.mark.parametrize("gap", [10.0, 20.0, 26.0, 30.0, 60.0])
@pytest.mark.parametrize("shape", [
    ([1] * 8, [30, 100, 7, 500, 64, 33, 2, 900], 8, 2, 128, 16), ([2, 1, 5], [40, 300, 77], 6, 2, 64, 24), ([1, 3], [50, 200], 4, 1, 256, 16),
])
def test_columns_of_small_weights(cuda, shape, gap, kind, dtype):
    new, kv, hq, hk, d, pt = shape
    q, k, v, table, cu, kv_len = make(cuda, 140, *shape, DT[dtype])
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    for s, (n, L) in enumerate(zip(new, kv)):            # an early key: its score is `gap` above, its values are 0 in half of the columns
        p = min(3, L - n)
        page = table[s, p // pt].item()
        k[page, :, p % pt] = 0
        k[page, :, p % pt, 0] = gap * d ** 0.5
        v[page, :, p % pt, ::2] = 0
    kp, vp, k, v = filled(k, v, kind)
    k, v = k.contiguous(), v.contiguous()
    out, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, max_new=max(new), return_lse=True)
    ref, rlse, tol, ltol = reference(q, k, v, table, new, kv)
    check(out, lse, (ref, rlse, tol + max(kv) * 2.0 ** -39 * v.abs().max(), ltol))
    if gap <= 10.0:                                      # weights that fp16 holds to 2^-11: as the reference alone
        check(out, lse, (ref, rlse, tol, ltol))

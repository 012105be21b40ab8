"""paged_quant_attention where every token has scales of its own: a lane of the rows kernel reads
scale bytes that other lanes copied, in the last tiles of a piece too, behind which no copies
follow.  Against float64 over the values held, as test_quant_attention_gpu.py; the same call gives
the same bits however often it runs."""
import pytest
import torch

import heteromm_b200 as hmm
from test_quant_attention_gpu import filled
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dtype", [("e4m3", "bf16"), ("int8", "fp16")])
@pytest.mark.parametrize("shape", [  # new, kv, hq, hk, d, pt
    ([1] * 40, [1 + 3 * i for i in range(40)], 8, 2, 128, 16),          # a tile or less a warp
    ([1] * 40, [100 + 11 * i for i in range(40)], 4, 4, 64, 16),
    ([2] * 24, [130 + 61 * i for i in range(24)], 8, 1, 256, 16),
    ([1] * 300, [1 + (37 * i) % 300 for i in range(300)], 4, 2, 128, 4),  # lists of several units a CTA
    ([1] * 30, [700 + 50 * i for i in range(30)], 6, 2, 96, 32),
    ([7] * 12, [7 + 90 * i for i in range(12)], 4, 1, 32, 16),
])
def test_every_token_its_own_scales(cuda, shape, kind, dtype):
    new, kv, hq, hk, d, pt = shape
    q, k, v, table, cu, kv_len = make(cuda, 70, new, kv, hq, hk, d, pt, DT[dtype])
    at = torch.arange(k.shape[0] * pt, device=cuda).view(-1, 1, pt, 1)
    group = torch.arange(d // 32, device=cuda).repeat_interleave(32)
    k *= 2.0 ** -((at * 5 + group * 3) % 7).to(k.dtype)                  # 2^-6 ... 1
    v *= 2.0 ** ((at * 7 + group * 5) % 13 - 6).to(v.dtype)              # 2^-6 ... 2^6
    kp, vp, k, v = filled(k, v, kind)
    ref = reference(q, k, v, table, new, kv)
    first = None
    for _ in range(20):
        out, lse = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, max_new=max(new), return_lse=True)
        if first is None:
            check(out, lse, ref)
            first = out, lse
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])

"""Bounded waits and units that take longer than their limit: the limit is for a step of the
work, not for all of it."""
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200 import _abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,rows", [(64, 256), (128, 256), (256, 128)])
def test_units_that_outlast_the_limit(cuda, d, rows):
    """A limit of 1 ms, and whole units of 2,048 key tiles, about 2 us each (a cache of 2^28
    tokens does the same to the default limit of 2 s)."""
    L, pt, n = 1 << 18, 128, 152 * rows
    g = torch.Generator(device=cuda).manual_seed(1)
    k = torch.randn((64, 1, pt, d), generator=g, device=cuda).to(torch.bfloat16)
    v = torch.randn((64, 1, pt, d), generator=g, device=cuda).to(torch.bfloat16)
    q = torch.randn((n, 1, d), generator=g, device=cuda).to(torch.bfloat16)
    table = (torch.arange(L // pt, dtype=torch.int32, device=cuda) % 64)[None].contiguous()
    cu, kv_len = torch.tensor([0, n], dtype=torch.int32, device=cuda), torch.tensor([L - 5], dtype=torch.int32, device=cuda)
    want = hmm.paged_attention(q, k, v, table, cu, kv_len)
    _abi.set_wait_limit_ns(1_000_000)
    try:
        got = hmm.paged_attention(q, k, v, table, cu, kv_len)
    finally:
        torch.cuda.synchronize()
        _abi.set_wait_limit_ns(-1)
    assert torch.equal(got, want)

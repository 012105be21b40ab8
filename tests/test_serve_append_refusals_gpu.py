"""Calls of paged_kv_append that are refused before anything is launched."""
import pytest
import torch

import heteromm_b200 as hmm
from test_serve_attention_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 32, 2), (8, 0, 2), (0, 0, 2)])
def test_an_empty_angle_table(cuda, shape):
    """Not the same as no table: nothing is stored unrotated."""
    q, k, v, table, cu, kv_len = make(cuda, 70, [2], [20], 4, 2, 64, 16, torch.bfloat16)
    kn, rope = torch.ones((2, 2, 64), dtype=torch.bfloat16, device=cuda), torch.zeros(shape, device=cuda)
    k0, v0 = k.clone(), v.clone()
    with pytest.raises(ValueError, match="rope"):
        hmm.paged_kv_append(q, kn, kn, k, v, table, cu, kv_len, rope)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    none = hmm.paged_kv_append(q[:0], kn[:0], kn[:0], k, v, table, torch.zeros_like(cu), kv_len, rope)   # no tokens to turn
    assert none.shape == (0, 4, 64)

"""Calls of paged_kv_append that are refused before anything is launched."""
import random

import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_INVALID, HmmError
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


def starts(t):
    """Byte ranges of a view's rows."""
    n, h, d = t.shape
    return {(i, j): t.data_ptr() + 2 * (i * t.stride(0) + j * t.stride(1)) for i in range(n) for j in range(h)}


def meet(a, b, same=False):
    size = 2 * a.shape[2]
    return any(abs(x - y) < size for i, x in starts(a).items() for j, y in starts(b).items() if not (same and i == j))


def test_out_anywhere_in_the_same_memory(cuda):
    """q, k, v and out as random views of one buffer: a call whose out shares a row with another's
    (but q's own, each at its place) is refused, the others give what separate arrays give."""
    rng = random.Random(5)
    d, hk, pt = 16, 1, 4
    rope = hmm.rope_table(16, d, device=cuda)
    table = torch.arange(4, dtype=torch.int32, device=cuda)[None]
    taken = kept = 0
    for _ in range(400):
        n, hq = rng.randint(1, 4), rng.randint(1, 3)
        cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        kv_len = torch.tensor([n + 3], dtype=torch.int32, device=cuda)
        flat = torch.randn(4096, device=cuda).to(torch.bfloat16)
        token = 8 * rng.randint(2, 16)

        def view(heads):
            t = token if rng.random() < 0.9 else 8 * rng.randint(0, 16)
            return flat.as_strided((n, heads, d), (t, 8 * rng.randint(0 if rng.random() < 0.1 else 2, 6), 1), 8 * rng.randint(0, 32))

        q, k, v = view(hq), view(hk), view(hk)
        out = q if rng.random() < 0.3 else view(hq)
        in_place = out.data_ptr() == q.data_ptr() and all(out.shape[i] == 1 or out.stride(i) == q.stride(i) for i in (0, 1))
        bad = meet(out, out, True) or (not in_place and meet(out, q)) or meet(out, k) or meet(out, v)
        kp, vp = (torch.zeros((4, hk, pt, d), dtype=torch.bfloat16, device=cuda) for _ in range(2))
        if bad:
            before = flat.clone()
            with pytest.raises(HmmError) as e:
                hmm.paged_kv_append(q, k, v, kp, vp, table, cu, kv_len, rope, out=out)
            assert e.value.status == HMM_ERR_INVALID and torch.equal(flat, before) and not kp.any()
            taken += 1
            continue
        k2, v2 = kp.clone(), vp.clone()
        want = hmm.paged_kv_append(q.clone(), k.clone(), v.clone(), k2, v2, table, cu, kv_len, rope)
        try:
            got = hmm.paged_kv_append(q, k, v, kp, vp, table, cu, kv_len, rope, out=out)
        except HmmError as e:     # rows of different token strides that interleave may be refused
            assert e.status == HMM_ERR_INVALID and n > 1 and len({x.stride(0) for x in (q, k, v, out)}) > 1
            continue
        assert torch.equal(got, want) and torch.equal(kp, k2) and torch.equal(vp, v2)
        kept += 1
    assert taken > 50 and kept > 50

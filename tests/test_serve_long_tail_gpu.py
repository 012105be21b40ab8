"""fp16 weights of a long flat tail behind a few dominant keys: their share must not be
lost to the type's smallest numbers.

A weight relative to the row's largest is held in fp16 times 2^14 (the rows kernel) or at
least 2^7 (the chunk kernel), so rounding it is off by at most half a step, 2^-11 of it, or
by half the smallest subnormal, 2^-25 of that factor: 2^-39 and 2^-32 of the largest weight.
The result is off by what these errors add to sum p v, by its own rounding, 2^-11 of it,
and by fp32: n / 16 = 2^13 sums of products (a tensor core's sum may truncate, 2^-23 each)
are off by 2^-10 of sum p |v| at most, the exponentials by less than 2^-16 of theirs.  A
thread adds to its sum of weights twice per 64 keys (rows kernel) or once (chunk kernel: per
half of a tile of 128), 2^12 or 2^11 times in 2^17 keys, each time off by 2^-24 of the sum:
that and lse by 2^-12 or 2^-13 of the sum."""
import pytest
import torch

import heteromm_b200 as hmm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,n_seq,hq", [("rows", 592, 1), ("rows", 1, 4), ("chunk", 148, 32), ("chunk", 148, 144),
                                             ("chunk", 2, 32)])
@pytest.mark.parametrize("nats", [18, 16.75])
def test_a_flat_tail(cuda, kernel, n_seq, hq, nats):
    """Keys 0, 16, 32, 48 and 128 score `nats` above 2^17 others, so that each warp's share of a
    unit has a dominant one; all sequences are the same pages."""
    L, d, pt = 1 << 17, 64, 128
    k = torch.zeros((L // pt, 1, pt, d), dtype=torch.float16, device=cuda)
    v = torch.zeros_like(k)
    v[..., :2] = 1.0
    v[..., 2] = torch.linspace(-1, 1, pt, device=cuda).to(torch.float16)
    for i in (0, 16, 32, 48, 128):
        k[i // pt, 0, i % pt, 0] = nats
        v[i // pt, 0, i % pt] = 0.0
        v[i // pt, 0, i % pt, 1] = -1.0
    q = torch.zeros((n_seq, hq, d), dtype=torch.float16, device=cuda)
    q[..., 0] = 1.0
    table = torch.arange(L // pt, dtype=torch.int32, device=cuda).repeat(n_seq, 1)
    cu = torch.arange(n_seq + 1, dtype=torch.int32, device=cuda)
    kv_len = torch.full((n_seq,), L, dtype=torch.int32, device=cuda)
    out, lse = hmm.paged_attention(q, k, v, table, cu, kv_len, scale=1.0, return_lse=True)
    p = (k.reshape(-1, d)[:, 0].double() - nats).exp()
    s, vv = p.sum(), v.reshape(-1, d).double()
    ref, mag = p @ vv / s, p @ vv.abs() / s
    off = torch.clamp(2.0 ** -11 * p, min=2.0 ** -39 if kernel == "rows" else 2.0 ** -32)
    total = 2.0 ** -12 if kernel == "rows" else 2.0 ** -13
    tol = (2.0 ** -11 + total) * ref.abs() + (1 + 2.0 ** -10) * (off @ vv.abs() / s) + (2.0 ** -10 + 2.0 ** -16) * mag + 2.0 ** -25
    worst = ((out.double() - ref).abs() / tol).amax()
    assert worst <= 1, (float(worst), out[0, 0, :3].tolist(), ref[:3].tolist())
    assert ((lse.double() - (nats + s.log())).abs() <= total + 2.0 ** -16).all()


def test_weights_do_not_overflow(cuda):
    """The largest weights that the chunk kernel makes, on values near the type's largest: from the
    second tile of keys on scores are 7.8 of log2 above the first's, which leaves its maximum."""
    n, d, pt = 700, 64, 16
    q = torch.ones((n, 1, d), dtype=torch.float16, device=cuda)
    k = torch.zeros((-(-n // pt) * pt, d), dtype=torch.float16, device=cuda)
    k[128:n] = 5.4 / d
    v = torch.full_like(k, 60000.0)
    table = torch.arange(len(k) // pt, dtype=torch.int32, device=cuda)[None]
    cu, kv_len = torch.tensor([0, n], dtype=torch.int32, device=cuda), torch.tensor([n], dtype=torch.int32, device=cuda)
    out, lse = hmm.paged_attention(q, k.view(-1, pt, d), v.view(-1, pt, d), table, cu, kv_len, scale=1.0, return_lse=True)
    # weights by half a step, the result too (16 at 60,000), and 1 for the fp32 sums
    assert (out.double() - 60000.0).abs().max() <= 60000 * 2.0 ** -11 + 16 + 1
    want = torch.logcumsumexp(k[:n].double().sum(1), 0)
    assert ((lse[:, 0].double() - want).abs() <= 2.0 ** -14).all()

"""The attention entry point at its ends: waits that run out, sequences that overlap, many
sequences, several host threads, the wrappers' refusals of device tensors."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200 import _abi
from heteromm_b200._abi import HMM_ERR_BOUNDS, HMM_ERR_TIMEOUT, HmmError
from test_serve_attention_gpu import check, make, reference, run_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,kv,hq,hk,d,max_new,must", [
    ([1, 1, 1], [500, 70, 2000], 16, 8, 128, 1, False),   # rows kernel: a tile or two a warp, which may
    ([1, 4], [3000, 4], 16, 8, 256, 0, False),            # have landed by the time they are asked for
    ([1] * 8, [40000] * 8, 2, 1, 128, 1, True),           # a long list from memory
    ([300, 40], [300, 900], 16, 8, 128, 0, True),         # both kernels, units cut
    ([700], [1500], 16, 8, 64, 0, True),
    ([2600, 2600], [2600, 3000], 16, 8, 128, 0, True),    # whole units
])
def test_a_wait_that_runs_out(cuda, new, kv, hq, hk, d, max_new, must):
    """A limit of 0: the first wait whose copy has not landed gives up, what is in flight
    lands, the call reports it, and the next call is as if nothing had been."""
    args = make(cuda, 40, new, kv, hq, hk, d, 16, torch.bfloat16)
    want = hmm.paged_attention(*args, max_new=max_new)
    for _ in range(3):
        _abi.set_wait_limit_ns(0)
        try:
            got = hmm.paged_attention(*args, max_new=max_new)
            assert not must and torch.equal(got, want)
        except HmmError as e:
            assert e.status == HMM_ERR_TIMEOUT
        finally:
            torch.cuda.synchronize()
            _abi.set_wait_limit_ns(-1)
        assert torch.equal(hmm.paged_attention(*args, max_new=max_new), want)


def test_overlapping_sequences_stay_inside(cuda):
    """A cu_new that goes to and fro: every second sequence is refused, the others overlap
    and are more work than the batch's tokens; nothing outside of the call's memory is
    written, and what follows is right."""
    n_seq, n_tok, hq, hk, d, pt = 64, 600, 2, 2, 64, 16
    q, k, v, table, cu, kv_len = make(cuda, 41, [n_tok] + [0] * (n_seq - 1), [n_tok] + [0] * (n_seq - 1), hq, hk, d, pt,
                                      torch.bfloat16)
    table[:] = table[0]
    kv_len[:] = n_tok
    back = torch.tensor([0 if i % 2 == 0 else n_tok for i in range(n_seq + 1)], dtype=torch.int32, device=cuda)
    need = _abi.load().hmm_paged_attention_workspace_size(n_seq, n_tok, hq, hk, d)
    ws = torch.full((need + (1 << 20),), 0x5a, dtype=torch.uint8, device=cuda)
    out = torch.full((n_tok + 64, hq, d), 7.0, dtype=torch.bfloat16, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    kc = _abi.PagedCache(k.data_ptr(), v.data_ptr(), k.shape[0], hk, pt, d, *k.stride()[:3], *v.stride()[:3],
                         _abi.HMM_DTYPE_BF16)
    b = _abi.PagedBatch(table.data_ptr(), n_seq, table.shape[1], back.data_ptr(), n_tok, kv_len.data_ptr())
    _abi.call("hmm_paged_attention", C.byref(kc), C.byref(b), q.data_ptr(), hq * d, d, hq, d ** -0.5, 1, 0, 0, 0,
              out.data_ptr(), None, status.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(HmmError) as e:
        _abi.call("hmm_status_read", status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert e.value.status == HMM_ERR_BOUNDS
    assert (ws[need:] == 0x5a).all() and (out[n_tok:] == 7.0).all()
    # (the overlapping sequences are the same one: their common rows are right)
    check(out, None, reference(q, k, v, table, [n_tok], [n_tok]))


@pytest.mark.parametrize("hq,hk,d", [(1, 1, 128), (4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("most", [40, 300, 900])
@pytest.mark.parametrize("window", [0, 50])
def test_many_sequences(cuda, hq, hk, d, most, window):
    """More than a warp's worth of sequences, with none, few and many new tokens, cut and
    whole units, one row block each and several."""
    rng = np.random.default_rng(most + d)
    n_seq = 75
    new = [int(x) for x in rng.integers(0, most, n_seq)]
    for i in range(0, n_seq, 5):
        new[i] = int(rng.integers(0, 2))
    new[33:66] = [0] * 33 if most == 300 else new[33:66]
    kv = [n + int(x) for n, x in zip(new, rng.integers(0, 200, n_seq))]
    run_case(cuda, 42, new, kv, hq, hk, d, 16, "bf16", pad=3, window=window, sinks=3 if window else 0)


def test_row_blocks_of_long_sequences_in_pieces(cuda):
    """Few units, cut into pieces that begin and end anywhere, beside units of one tile."""
    run_case(cuda, 43, [256, 1, 600, 0, 2, 30], [6000, 9, 5001, 4, 800, 30], 8, 1, 128, 16, "fp16")
    run_case(cuda, 43, [500] + [20] * 40, [4000] + [20] * 40, 1, 1, 64, 64, "bf16", window=700, sinks=5)


def test_a_batch_of_thousands(cuda):
    new, kv = [1, 0, 1, 20] * 500, [40, 7, 3, 20] * 500
    run_case(cuda, 44, new, kv, 2, 1, 64, 16, "bf16")


def test_nothing_to_attend_to(cuda):
    """No tokens, no sequences, no room: outputs as the formula has them, or untouched."""
    q, k, v, table, cu, kv_len = make(cuda, 49, [3, 2], [20, 9], 4, 2, 64, 16, torch.bfloat16)
    none = torch.zeros_like(cu)
    assert hmm.paged_attention(q[:0], k, v, table, none, kv_len).shape == (0, 4, 64)
    out = torch.full_like(q, 5.0)
    hmm.paged_attention(q, k, v, table, none, kv_len, out=out)                      # no new tokens
    hmm.paged_attention(q, k, v, table[:0], cu[:1], kv_len[:0], out=out)            # no sequences
    assert (out == 5.0).all()
    got, lse = hmm.paged_attention(q, k, v, table[:, :0].contiguous(), cu, torch.zeros_like(kv_len), return_lse=True)
    assert (got == 0).all() and (lse == -np.inf).all()                              # nothing cached
    assert hmm.paged_kv_append(q[:0], k[:0, :, 0], v[:0, :, 0], k, v, table, none, kv_len).shape == (0, 4, 64)


def test_a_thousand_sequences(cuda):
    new = [1] * 1000 + [300] + [0] * 30
    kv = [(37 * i) % 90 + 1 for i in range(1000)] + [500] + [3] * 30
    run_case(cuda, 50, new, kv, 4, 1, 128, 16, "bf16")


def test_two_threads_on_two_streams(cuda):
    cases = [make(cuda, 45 + i, new, kv, 8, 2, 128, 16, torch.bfloat16)
             for i, (new, kv) in enumerate((([300, 2], [900, 700]), ([1] * 20, list(range(50, 1050, 50)))))]
    want = [hmm.paged_attention(*c, max_new=0) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(c, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    if not torch.equal(hmm.paged_attention(*c), w):
                        bad.append("differs")
        except Exception as e:   # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_wrappers_refuse(cuda):
    q, k, v, table, cu, kv_len = make(cuda, 46, [2, 3], [20, 30], 4, 2, 64, 16, torch.bfloat16)

    def bad(exc, **kw):
        a = dict(q=q, k_pages=k, v_pages=v, page_table=table, cu_new=cu, kv_len=kv_len)
        a.update(kw)
        with pytest.raises(exc):
            hmm.paged_attention(**a)

    bad(TypeError, q=q.half())
    bad(TypeError, k_pages=k.float(), v_pages=v.float())
    bad(ValueError, v_pages=v[:-1])
    bad(ValueError, v_pages=v.half())
    bad(ValueError, q=q[..., :32])
    bad(ValueError, q=q[0])
    bad(ValueError, q=q.cpu())
    bad(ValueError, k_pages=k.permute(0, 1, 3, 2), v_pages=v.permute(0, 1, 3, 2), q=torch.cat([q] * 1)[..., :16])
    bad(TypeError, page_table=table.long())
    bad(ValueError, page_table=table[0])
    bad(ValueError, page_table=table.T)
    bad(ValueError, cu_new=cu[:-1])
    bad(ValueError, kv_len=kv_len.cpu())
    bad(ValueError, kv_len=kv_len[:1])
    bad(ValueError, out=torch.empty_like(q)[:-1])
    bad(TypeError, out=torch.empty_like(q).half())
    bad(ValueError, status=torch.zeros(1, dtype=torch.int32))
    bad(TypeError, status=torch.zeros(1, dtype=torch.int64, device=cuda))
    bad(HmmError, q=q[:, :3])
    bad(HmmError, window=-1)
    bad(HmmError, causal=False, window=5)
    bad(HmmError, q=torch.zeros(q.numel() + 4, dtype=q.dtype, device=cuda)[4:].view(q.shape))
    bad(HmmError, k_pages=k[:0], v_pages=v[:0])
    kn, qn = k[:5, :, 0], q[:, :2]
    for exc, kw in ((ValueError, dict(k=kn[:4])), (TypeError, dict(v=kn.half())), (ValueError, dict(q=q[:4])),
                    (TypeError, dict(q_weight=torch.ones(64, dtype=torch.float64, device=cuda))),
                    (ValueError, dict(k_weight=torch.ones(32, device=cuda))),
                    (ValueError, dict(rope=torch.ones(8, 64, device=cuda))),
                    (TypeError, dict(rope=torch.ones(8, 32, 2, device=cuda).half())),
                    (TypeError, dict(positions=torch.zeros(5, dtype=torch.int64, device=cuda))),
                    (ValueError, dict(positions=torch.zeros(4, dtype=torch.int32, device=cuda)))):
        a = dict(q=qn, k=kn, v=kn, k_pages=k, v_pages=v, page_table=table, cu_new=cu, kv_len=kv_len)
        a.update(kw)
        with pytest.raises(exc):
            hmm.paged_kv_append(**a)


@pytest.mark.parametrize("d,pt,dtype", [(256, 16, "bf16"), (200, 8, "fp16"), (136, 128, "bf16")])
@pytest.mark.parametrize("new,kv,hq,hk", [
    ([700, 1, 130, 0, 33], [900, 50, 4000, 7, 33], 6, 2),     # cut units
    ([1500, 800], [1500, 2000], 16, 4),                       # whole ones
    ([128, 129, 127, 17, 16], [128, 300, 127, 17, 400], 1, 1),
])
@pytest.mark.parametrize("window", [0, 300])
def test_wide_heads(cuda, d, pt, dtype, new, kv, hq, hk, window):
    """Heads of more than 128 values: units of 128 rows."""
    run_case(cuda, 47, new, kv, hq, hk, d, pt, dtype, pad=2, window=window, sinks=5 if window else 0)


def test_wide_heads_wait(cuda):
    args = make(cuda, 48, [900, 300], [900, 1200], 8, 2, 256, 16, torch.float16)
    want = hmm.paged_attention(*args)
    _abi.set_wait_limit_ns(0)
    try:
        with pytest.raises(HmmError) as e:
            hmm.paged_attention(*args)
        assert e.value.status == HMM_ERR_TIMEOUT
    finally:
        torch.cuda.synchronize()
        _abi.set_wait_limit_ns(-1)
    assert torch.equal(hmm.paged_attention(*args), want)

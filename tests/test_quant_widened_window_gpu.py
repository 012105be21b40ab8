"""paged_quant_attention where keys are widened into the workspace and a window leaves most of them
out: pages behind every row's window stay unwritten there, those of the first tokens are kept.
Through the C entry, over a workspace that is NaN throughout.  That keys were widened, and that
others were not, is seen from the workspace, which holds their rows or does not."""
import ctypes as C

import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import (HMM_DTYPE_BF16, HMM_DTYPE_E4M3, HMM_DTYPE_F16, HMM_DTYPE_I8, HMM_OK, PagedBatch, PagedQuant)
from test_quant_attention_gpu import filled, raw
from test_serve_attention_gpu import DT, check, make, reference

pytestmark = pytest.mark.gpu

NAN = float("nan")


def call(q, kp, vp, table, cu, kv_len, scale, causal=True, window=0, sinks=0, max_new=0, fill=255):
    """(out, lse, status, workspace) of hmm_paged_quant_attention, the workspace's bytes being `fill` before."""
    lib, (n, hq, d), (pages, hk, pt, _) = hmm.load(), q.shape, kp.shape
    cache = PagedQuant(kp.data_ptr(), vp.data_ptr(), pages, hk, pt, d, kp.stride(0), kp.stride(1), vp.stride(0), vp.stride(1),
                       HMM_DTYPE_I8 if kp.dtype == torch.int8 else HMM_DTYPE_E4M3)
    batch = PagedBatch(table.data_ptr(), table.shape[0], table.shape[1], cu.data_ptr(), n, kv_len.data_ptr())
    size = lib.hmm_paged_quant_attention_workspace_size(table.shape[0], n, hq, hk, d, table.shape[1] * pt, max_new)
    ws = torch.full((size,), fill, dtype=torch.uint8, device=q.device)
    out = torch.full_like(q, 9.0)
    lse = torch.full((n, hq), 9.0, device=q.device)
    status = torch.zeros(1, dtype=torch.int32, device=q.device)
    r = lib.hmm_paged_quant_attention(C.byref(cache), C.byref(batch), HMM_DTYPE_BF16 if q.dtype == torch.bfloat16 else HMM_DTYPE_F16,
                                      q.data_ptr(), hq * d, d, hq, scale, int(causal), window, sinks, max_new, out.data_ptr(),
                                      lse.data_ptr(), status.data_ptr(), ws.data_ptr(), size,
                                      torch.cuda.current_stream().cuda_stream)
    assert r == HMM_OK, lib.hmm_last_error()
    return out, lse, status, ws


def held(ws, row):
    """Whether the workspace has this row's first 32 values somewhere."""
    n = ws.numel() // 64 * 64
    return bool((ws[:n].view(torch.int16).view(-1, 32) == row[:32].contiguous().view(torch.int16)).all(-1).any())


CASES = [  # new, kv, hq, hk, d, pt, window, sinks: products enough to widen, by 8 heads, 18 tiles of keys and 29 blocks of rows
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 64, 16, 2000, 0),
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 64, 16, 2000, 5),
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 128, 16, 2000, 133),     # first tokens end within the second page there
    ([700, 1, 220], [6000, 300, 2900], 64, 8, 96, 64, 2000, 1),
    ([350, 500, 90], [6001, 4000, 2900], 64, 8, 256, 16, 2000, 40),
    ([940], [7013], 64, 8, 128, 128, 2050, 4),                         # one sequence
]


@pytest.mark.parametrize("kind,dtype", [("e4m3", "bf16"), ("int8", "fp16")])
@pytest.mark.parametrize("case", CASES)
def test_window(cuda, case, kind, dtype):
    new, kv, hq, hk, d, pt, window, sinks = case
    pad = 20
    q, k, v, table, cu, kv_len = make(cuda, 100, new, kv, hq, hk, d, pt, DT[dtype], pad=pad)
    kp, vp, k, v = filled(k, v, kind)
    k, v = k.contiguous(), v.contiguous()
    ref = reference(q, k, v, table, new, kv, window=window, sinks=sinks)
    ts = table.clone()
    for s, (n, L) in enumerate(zip(new, kv)):       # pages that no row sees are gone
        first = max(0, L - n - window + 1)
        for i in range(-(-sinks // pt), first // pt):
            table[s, i] = -1 if i % 2 else 1 << 30
    out, lse, status, ws = call(q, kp, vp, table, cu, kv_len, d ** -0.5, window=window, sinks=sinks)
    assert status.item() == 0
    check(out, lse, ref)
    assert (out[sum(new):] == 9.0).all() and (lse[sum(new):] == 9.0).all()
    row = lambda p: v[ts[0, p // pt].item(), hk - 1, p % pt]  # noqa: E731
    first = kv[0] - new[0] - window + 1
    assert held(ws, row(kv[0] - 1)) and held(ws, row(first)), "its keys were not widened"
    assert not held(ws, row(first - 1)) and not held(ws, row(first // 2 + 100))
    if sinks:
        assert held(ws, row(0)) and held(ws, row(sinks - 1)) and not held(ws, row(sinks))
    again = hmm.paged_quant_attention(q, kp, vp, table, cu, kv_len, window=window, sinks=sinks)
    assert torch.equal(again[:sum(new)], out[:sum(new)]), "the same call, the same bits"


def test_values_that_are_not_finite(cuda):
    """NaN groups behind the window, between it and the first tokens and behind the end reach
    nothing; one within some rows' windows, and one of a first token, those rows alone."""
    new, kv, hq, hk, d, pt, window, sinks = [700, 1, 220], [6000, 300, 2900], 64, 8, 64, 16, 2000, 5
    q, k, v, table, cu, kv_len = make(cuda, 101, new, kv, hq, hk, d, pt, torch.bfloat16, pad=20)
    kp, vp, k, v = filled(k, v, "e4m3")
    k, v = k.contiguous(), v.contiguous()

    def bad(pages, values, p, head, group):
        page = table[0, p // pt].item()
        codes, scales = raw(pages)
        codes[page, head, p % pt, 32 * group:32 * group + 32], scales[page, head, p % pt, group] = 0, 255
        values[page, head, p % pt, 32 * group:32 * group + 32] = NAN

    first = kv[0] - new[0] - window + 1
    for p in (sinks, 100, first - 1):
        bad(vp, v, p, 1, 0)
        bad(kp, k, p, 1, 1)
    out, lse, status, ws = call(q, kp, vp, table, cu, kv_len, d ** -0.5, window=window, sinks=sinks)
    assert status.item() == 0 and torch.isfinite(out).all() and held(ws, v[table[0, first // pt].item(), 7, first % pt])
    check(out, lse, reference(q, k, v, table, new, kv, window=window, sinks=sinks))
    bad(vp, v, first + 300, 2, 1)                    # the first 301 rows' windows
    out, lse, status, _ = call(q, kp, vp, table, cu, kv_len, d ** -0.5, window=window, sinks=sinks)
    check(out, lse, reference(q, k, v, table, new, kv, window=window, sinks=sinks))
    bad(vp, v, 2, 3, 0)
    bad(kp, k, 4, 4, 1)
    out, lse, status, _ = call(q, kp, vp, table, cu, kv_len, d ** -0.5, window=window, sinks=sinks)
    check(out, lse, reference(q, k, v, table, new, kv, window=window, sinks=sinks))
    assert status.item() == 0


@pytest.mark.parametrize("causal", [True, False])
def test_no_window(cuda, causal):
    """The same over a NaN workspace without a window: all keys are widened, and nothing of what lay
    behind a sequence's end there is read."""
    new, kv, hq, hk, d, pt = [700, 1, 221], [1300, 300, 1101], 64, 8, 64, 16
    q, k, v, table, cu, kv_len = make(cuda, 102, new, kv, hq, hk, d, pt, torch.float16)
    kp, vp, k, v = filled(k, v, "int8")
    table = torch.nn.functional.pad(table, (0, 100), value=-1)
    out, lse, status, ws = call(q, kp, vp, table, cu, kv_len, 0.1, causal=causal)
    assert status.item() == 0 and held(ws, v[table[0, 0].item(), 0, 0]) and held(ws, v[table[2, 1100 // pt].item(), 7, 1100 % pt])
    check(out, lse, reference(q, k.contiguous(), v.contiguous(), table, new, kv, causal=causal, scale=0.1))

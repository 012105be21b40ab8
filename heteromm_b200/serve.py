"""Torch-facing wrappers of the serving entry points: filling a paged cache of
several KV heads, attending over it with ragged chunks of new tokens, and
managing its pages.

A cache is two page arrays `k_pages`, `v_pages` [n_pages, n_kv_heads, page_tokens, D]
of bf16 or fp16 (int16 is read as bf16 bit patterns, as elsewhere in the package),
or [n_pages, page_tokens, D] for one head.  Any page / head / token strides that are
multiples of 8 elements do, with the last dimension contiguous: token-major pages are
`pages.transpose(1, 2)`, interleaved ones `both[:, 0]` and `both[:, 1]`.

A batch is `page_table` [n_seq, pages_per_seq] int32, `cu_new` [n_seq + 1] int32 (the
rows of each sequence's new tokens in the packed arrays) and `kv_len` [n_seq] int32
(cached tokens, the new ones among them).  All of it is read on the device; rows that
no sequence owns are left as they are.

Every call runs on the current stream of its tensors' device.  With `status` (an int32
device tensor that the caller zeroes) it does not wait: flags of bad page-table
entries, lengths, positions or sequence numbers and of too few free pages gather in it,
and check_status(status) raises for them later; without it the call waits and raises
HmmError itself, so inside a stream capture a status is needed.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._abi import HMM_DTYPE_BF16, HMM_DTYPE_F16, HMM_DTYPE_F32, PageStore, PagedBatch, PagedCache, \
    PagedState, call, load

_DTYPES = {torch.bfloat16: HMM_DTYPE_BF16, torch.int16: HMM_DTYPE_BF16,
           torch.float16: HMM_DTYPE_F16}


def _tensor(t, name: str, dtype, device, shape=None, contiguous: bool = True):
    """Checks one argument; `device` None accepts any CUDA device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the others are on {device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _four(pages: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(pages, torch.Tensor) or not pages.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if pages.dim() == 3:
        pages = pages.unsqueeze(1)
    if pages.dim() != 4:
        raise ValueError(f"{name} must be [n_pages, n_kv_heads, page_tokens, D]")
    if pages.dtype not in _DTYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or int16 (bf16 bits), got {pages.dtype}")
    if pages.stride(3) != 1 and pages.shape[3] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return pages


def _cache(k_pages: torch.Tensor, v_pages: torch.Tensor):
    """(device, dtype, n_kv_heads, page_tokens, D, PagedCache)."""
    k, v = _four(k_pages, "k_pages"), _four(v_pages, "v_pages")
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("k_pages and v_pages differ in shape, dtype or device")
    n, h, pt, d = k.shape
    ks, vs = k.stride(), v.stride()
    return k.device, k.dtype, h, pt, d, PagedCache(
        k.data_ptr(), v.data_ptr(), n, h, pt, d, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        _DTYPES[k.dtype])


def _batch(page_table, cu_new, kv_len, n_tokens: int, device) -> PagedBatch:
    _tensor(page_table, "page_table", torch.int32, device)
    if page_table.dim() != 2:
        raise ValueError("page_table must be [n_seq, pages_per_seq]")
    n_seq, pps = page_table.shape
    _tensor(cu_new, "cu_new", torch.int32, device, (n_seq + 1,))
    _tensor(kv_len, "kv_len", torch.int32, device, (n_seq,))
    return PagedBatch(page_table.data_ptr(), n_seq, pps, cu_new.data_ptr(), n_tokens,
                      kv_len.data_ptr())


def _rows(t, name: str, dtype, device, n_tokens: int, heads: int, d: int):
    """(pointer, token stride, head stride) of packed rows [n_tokens, heads, D]."""
    _tensor(t, name, dtype, device, (n_tokens, heads, d), contiguous=False)
    if t.stride(2) != 1 and d > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _run(device, status, issue):
    """issue(status pointer, stream) on the current stream of `device`; without a
    status waits for it and raises."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _run(device, status, issue)
    stream = torch.cuda.current_stream().cuda_stream
    if status is not None:
        _tensor(status, "status", torch.int32, device)
        if status.numel() < 1:
            raise ValueError("status must hold an int32")
        issue(status.data_ptr(), stream)
        return
    own = torch.zeros(1, dtype=torch.int32, device=device)
    issue(own.data_ptr(), stream)
    call("hmm_status_read", own.data_ptr(), stream)


def rope_table(n_pos: int, rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """[n_pos, rotary_dim / 2, 2] fp32 (cos, sin) of p * theta^(-2i / rotary_dim), the
    angles in 64 bits: laid out once, for paged_kv_append."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * theta ** (-2.0 * i / rotary_dim)[None, :]
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous().to(device)


def paged_kv_append(q, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                    v_pages: torch.Tensor, page_table: torch.Tensor, cu_new: torch.Tensor,
                    kv_len: torch.Tensor, rope: torch.Tensor | None = None, *, q_weight=None,
                    k_weight=None, eps: float = 1e-6, interleaved: bool = False, positions=None,
                    out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """The step before attention in one pass: RMS norm of each query and key head (with
    q_weight, k_weight [D], fp32 or the cache's type), rotation of their first
    2 * rope.shape[1] values by rope [n_pos, pairs, 2] fp32 (cos, sin), and the store of
    keys and values into the cache.  Returns the queries (in `out`, which may be q).

    q [n_tokens, n_heads, D] (or None: keys and values alone), k, v
    [n_tokens, n_kv_heads, D], views of one projection included.  Pairs are halves
    (i, i + pairs), or neighbours with `interleaved`; the angle's row is the token's
    position, or positions [n_tokens] int32."""
    device, dtype, hk, _, d, cache = _cache(k_pages, v_pages)
    n_tokens = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else -1
    kp = _rows(k, "k", dtype, device, n_tokens, hk, d)
    vp = _rows(v, "v", dtype, device, n_tokens, hk, d)
    heads, qp, op = 0, (None, 0, 0), (None, 0, 0)
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must be [n_tokens, n_heads, D]")
        heads = q.shape[1]
        qp = _rows(q, "q", dtype, device, n_tokens, heads, d)
        if out is None:
            out = torch.empty((n_tokens, heads, d), dtype=dtype, device=device)
        op = _rows(out, "out", dtype, device, n_tokens, heads, d)
    batch = _batch(page_table, cu_new, kv_len, n_tokens, device)
    wdt, wptr = -1, [None, None]
    for i, (w, name) in enumerate(((q_weight, "q_weight"), (k_weight, "k_weight"))):
        if w is None:
            continue
        if isinstance(w, torch.Tensor) and w.dtype != dtype and w.dtype != torch.float32:
            raise TypeError(f"{name} must be float32 or {dtype}, got {w.dtype}")
        _tensor(w, name, w.dtype if isinstance(w, torch.Tensor) else dtype, device, (d,))
        this = HMM_DTYPE_F32 if w.dtype == torch.float32 else _DTYPES[dtype]
        if wdt not in (-1, this):
            raise TypeError("q_weight and k_weight must have the same dtype")
        wdt, wptr[i] = this, w.data_ptr()
    rp, n_pos, rotary = None, 0, 0
    if rope is not None:
        _tensor(rope, "rope", torch.float32, device)
        if rope.dim() != 3 or rope.shape[2] != 2:
            raise ValueError("rope must be [n_pos, pairs, 2]")
        rp, n_pos, rotary = rope.data_ptr(), rope.shape[0], 2 * rope.shape[1]
    if positions is not None:
        _tensor(positions, "positions", torch.int32, device, (n_tokens,))

    _run(device, status, lambda st, stream: call(
        "hmm_paged_kv_append", C.byref(cache), C.byref(batch), qp[0], qp[1], qp[2], heads, *kp, *vp,
        wptr[0], wptr[1], wdt, eps, rp, n_pos, rotary, int(interleaved),
        None if positions is None else positions.data_ptr(), op[0], op[1], op[2], st, stream))
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, cu_new: torch.Tensor, kv_len: torch.Tensor, *,
                    causal: bool = True, window: int = 0, sinks: int = 0,
                    scale: float | None = None, max_new: int = 0, return_lse: bool = False,
                    out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """Attention of the batch's new tokens over the cache, which holds them already
    (paged_kv_append): out [n_tokens, n_heads, D] of q's dtype, and with return_lse the
    log of each row's sum of exponentials [n_tokens, n_heads] fp32.

    A token at position p sees keys i <= p (all with causal=False) of its sequence; with a
    window only i > p - window, and i < sinks.  One that sees none gives zeros and -inf.
    q [n_tokens, n_heads, D]; query head h reads KV head h // (n_heads // n_kv_heads).
    scale defaults to D ** -0.5.  max_new, a bound on the new tokens of any sequence,
    helps to choose the kernel (decoding: 1); results do not depend on it."""
    device, dtype, hk, _, d, cache = _cache(k_pages, v_pages)
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [n_tokens, n_heads, D]")
    n_tokens, heads = q.shape[:2]
    qp = _rows(q, "q", dtype, device, n_tokens, heads, d)
    batch = _batch(page_table, cu_new, kv_len, n_tokens, device)
    if out is None:
        out = torch.empty((n_tokens, heads, d), dtype=dtype, device=device)
    else:
        _tensor(out, "out", dtype, device, (n_tokens, heads, d))
    lse = torch.empty((n_tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    ws = torch.empty(load().hmm_paged_attention_workspace_size(
        batch.n_seq, n_tokens, heads, hk, d), dtype=torch.uint8, device=device)
    _run(device, status, lambda st, stream: call(
        "hmm_paged_attention", C.byref(cache), C.byref(batch), *qp, heads,
        d ** -0.5 if scale is None else scale, int(causal), window, sinks, max_new, out.data_ptr(),
        None if lse is None else lse.data_ptr(), st, ws.data_ptr(), ws.numel(), stream))
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ pages


def _store(k_pages: torch.Tensor, v_pages: torch.Tensor) -> tuple:
    """(device, PageStore) of page arrays [(n_layers,) n_pages, ...]; a page (all but the
    leading dimensions) must be one block of memory."""
    views = []
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if t.dim() not in (3, 4, 5):
            raise ValueError(f"{name} must be [n_pages, n_kv_heads, page_tokens, D], with a "
                             "leading dimension of layers or not")
        layers, rest = (t.shape[0], t.shape[2:]) if t.dim() == 5 else (1, t.shape[1:])
        strides = t.stride()[2:] if t.dim() == 5 else t.stride()[1:]
        need = 1
        for n, s in sorted(zip(rest, strides), key=lambda x: (x[1], x[0])):
            if n != 1 and s != need:
                raise ValueError(f"{name}: a page must be one block of memory")
            need *= n
        b = t.element_size()
        page = t.stride(1 if t.dim() == 5 else 0) * b
        views.append((t.data_ptr(), page, t.stride(0) * b if t.dim() == 5 else 0, need * b, layers))
    if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or \
            k_pages.device != v_pages.device:
        raise ValueError("k_pages and v_pages differ in shape, dtype or device")
    (kp, kps, kls, nbytes, layers), (vp, vps, vls, _, _) = views
    n_pages = k_pages.shape[1 if k_pages.dim() == 5 else 0]
    return k_pages.device, PageStore(kp, vp, n_pages, nbytes, layers, kps, kls, vps, vls)


def _state(page_table, refs, kv_len, out, device):
    """(PagedState, [new page_table, refs, kv_len], workspace)."""
    _tensor(page_table, "page_table", torch.int32, device)
    if page_table.dim() != 2:
        raise ValueError("page_table must be [n_seq, pages_per_seq]")
    device = page_table.device
    n_seq, pps = page_table.shape
    _tensor(refs, "refs", torch.int32, device)
    if refs.dim() != 1:
        raise ValueError("refs must be [n_pages]")
    old = [page_table, refs]
    if kv_len is not None:
        _tensor(kv_len, "kv_len", torch.int32, device, (n_seq,))
        old.append(kv_len)
    if out is None:
        new = [torch.empty_like(t) for t in old]
    else:
        new = list(out)
        if len(new) != len(old):
            raise ValueError(f"out must hold {len(old)} tensors")
        for t, o, name in zip(new, old, ("page_table", "refs", "kv_len")):
            _tensor(t, f"out {name}", torch.int32, device, tuple(o.shape))
    ptr = [t.data_ptr() for t in old] + ([0] if kv_len is None else [])
    nptr = [t.data_ptr() for t in new] + ([0] if kv_len is None else [])
    ws = torch.empty(load().hmm_paged_state_workspace_size(n_seq, refs.shape[0]), dtype=torch.uint8,
                     device=device)
    return PagedState(*ptr, *nptr, n_seq, pps, refs.shape[0]), new, ws


def _ids(t, name: str, device, n=None) -> int:
    _tensor(t, name, torch.int32, device)
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be a vector" + ("" if n is None else f" of {n}"))
    return t.shape[0]


def paged_copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor,
                     dst: torch.Tensor, *, status: torch.Tensor | None = None) -> None:
    """Copies page src[i] to page dst[i] (int32) of K and V, in every layer of
    [n_layers, n_pages, n_kv_heads, page_tokens, D] arrays; a pair with a negative entry
    is skipped.  Nothing is copied, and BOUNDS raised, if a page is out of range, a dst is
    listed twice or is another pair's src."""
    device, store = _store(k_pages, v_pages)
    n = _ids(src, "src", device)
    _ids(dst, "dst", device, n)
    ws = torch.empty(1, dtype=torch.int32, device=device)
    _run(device, status, lambda st, stream: call(
        "hmm_paged_copy_pages", C.byref(store), src.data_ptr(), dst.data_ptr(), n, st,
        ws.data_ptr(), 4, stream))


def paged_free(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               seqs: torch.Tensor, *, out=None, status: torch.Tensor | None = None):
    """Frees the sequences of `seqs` (int32; one listed twice is freed once): their pages
    lose a reference each, their rows become -1 and their lengths 0.  Returns the new
    (page_table, refs, kv_len): new tensors, or `out`, which may be the old ones."""
    state, new, ws = _state(page_table, refs, kv_len, out, None)
    n = _ids(seqs, "seqs", page_table.device)
    _run(page_table.device, status, lambda st, stream: call(
        "hmm_paged_free", C.byref(state), seqs.data_ptr(), n, st, ws.data_ptr(), ws.numel(), stream))
    return tuple(new)


def paged_fork(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               src: torch.Tensor, dst: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               *, out=None, status: torch.Tensor | None = None):
    """Forks sequence src[i] into the empty row dst[i]: full pages are shared, a partly
    filled last page is copied into the lowest free one (in every layer of
    [n_layers, n_pages, ...] arrays).  Returns the new (page_table, refs, kv_len) as
    paged_free does.  A request that cannot be met as a whole changes nothing."""
    device, store = _store(k_pages, v_pages)
    state, new, ws = _state(page_table, refs, kv_len, out, device)
    n = _ids(src, "src", device)
    _ids(dst, "dst", device, n)
    pt = k_pages.shape[-2]
    _run(device, status, lambda st, stream: call(
        "hmm_paged_fork", C.byref(state), C.byref(store), pt, src.data_ptr(), dst.data_ptr(), n, st,
        ws.data_ptr(), ws.numel(), stream))
    return tuple(new)


def paged_grow(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               n_new: torch.Tensor, page_tokens: int, *, out=None,
               status: torch.Tensor | None = None):
    """Makes room for n_new[s] more tokens of every sequence: entries of the pages they
    touch that hold none get the lowest free pages, in row order.  Returns the new
    (page_table, refs, kv_len + n_new) as paged_free does."""
    state, new, ws = _state(page_table, refs, kv_len, out, None)
    _ids(n_new, "n_new", page_table.device, page_table.shape[0])
    _run(page_table.device, status, lambda st, stream: call(
        "hmm_paged_grow", C.byref(state), page_tokens, n_new.data_ptr(), st, ws.data_ptr(),
        ws.numel(), stream))
    return tuple(new)


def paged_compact(page_table: torch.Tensor, refs: torch.Tensor, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, *, out=None, status: torch.Tensor | None = None):
    """Moves the live pages (refs != 0) to the front of the cache, each at most once: the
    k-th live page behind the front goes to the k-th free one in it.  Returns
    (page_table, refs, live [1] int32); `out` holds the first two.  Page numbers kept
    elsewhere than in page_table do not follow."""
    device, store = _store(k_pages, v_pages)
    state, new, ws = _state(page_table, refs, None, out, device)
    live = torch.empty(1, dtype=torch.int32, device=device)
    _run(device, status, lambda st, stream: call(
        "hmm_paged_compact", C.byref(state), C.byref(store), live.data_ptr(), st, ws.data_ptr(),
        ws.numel(), stream))
    return (*new, live)

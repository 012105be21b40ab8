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
import functools

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream
from torch.cuda import current_device as _current_device

from ._abi import HMM_DTYPE_BF16, HMM_DTYPE_F16, HMM_DTYPE_F32, PageStore, PagedBatch, PagedCache, \
    PagedState, call, load

_DTYPES = {torch.bfloat16: HMM_DTYPE_BF16, torch.int16: HMM_DTYPE_BF16,
           torch.float16: HMM_DTYPE_F16}
_i32 = torch.int32

# These calls are issued once per layer and token, so the checks of a valid call are one
# expression; what is wrong is worked out only for the message.


def _refuse(t, name: str, dtype, dev: int, shape) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on cuda:{t.get_device()}, the others are on cuda:{dev}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _tensor(t, name: str, dtype, dev: int, shape=None) -> int:
    """The pointer of a contiguous tensor of this dtype, device and shape."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and
            (shape is None or t.shape == shape) and t.is_contiguous()):
        _refuse(t, name, dtype, dev, shape)
    return t.data_ptr()


def _rows(t, name: str, dtype, dev: int, shape):
    """(pointer, token stride, head stride) of packed rows [n_tokens, heads, D]."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and
            t.shape == shape):
        _refuse(t, name, dtype, dev, shape)
    st = t.stride()
    if st[2] != 1 and shape[2] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t.data_ptr(), st[0], st[1]


def _four(pages, name: str) -> torch.Tensor:
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


def _cache(k_pages, v_pages):
    """(device index, dtype, n_kv_heads, D, PagedCache)."""
    k, v = _four(k_pages, "k_pages"), _four(v_pages, "v_pages")
    shape, dtype, dev = k.shape, k.dtype, k.get_device()
    if v.shape != shape or v.dtype is not dtype or v.get_device() != dev:
        raise ValueError("k_pages and v_pages differ in shape, dtype or device")
    n, h, pt, d = shape
    ks, vs = k.stride(), v.stride()
    return dev, dtype, h, d, PagedCache(k.data_ptr(), v.data_ptr(), n, h, pt, d, ks[0], ks[1], ks[2],
                                        vs[0], vs[1], vs[2], _DTYPES[dtype])


def _table(page_table, dev: int):
    """(pointer, n_seq, pages_per_seq)."""
    p = _tensor(page_table, "page_table", _i32, dev)
    if page_table.dim() != 2:
        raise ValueError("page_table must be [n_seq, pages_per_seq]")
    return p, *page_table.shape


def _batch(page_table, cu_new, kv_len, n_tokens: int, dev: int) -> PagedBatch:
    p, n_seq, pps = _table(page_table, dev)
    return PagedBatch(p, n_seq, pps, _tensor(cu_new, "cu_new", _i32, dev, (n_seq + 1,)), n_tokens,
                      _tensor(kv_len, "kv_len", _i32, dev, (n_seq,)))


def _on_device(f):
    """Runs the call with the device of its first tensor as the current one."""
    @functools.wraps(f)
    def g(*args, **kw):
        for t in args or kw.values():
            if isinstance(t, torch.Tensor):
                dev = t.get_device()   # -1 for a CPU tensor, which f refuses
                if dev >= 0 and dev != _current_device():
                    with torch.cuda.device(dev):
                        return f(*args, **kw)
                break
        return f(*args, **kw)
    return g


def _status(status, dev: int):
    """(the status tensor of the call, its pointer, whether the call waits for it)."""
    if status is None:
        status = torch.zeros(1, dtype=_i32, device=dev)
        return status, status.data_ptr(), True
    if not (isinstance(status, torch.Tensor) and status.dtype is _i32 and status.get_device() == dev and
            status.numel() > 0):
        _refuse(status, "status", _i32, dev, (1,))
    return status, status.data_ptr(), False


def _wait(own, stream: int) -> None:
    call("hmm_status_read", own.data_ptr(), stream)


@functools.lru_cache(maxsize=256)
def _attention_workspace(dev: int, *sizes) -> int:
    return load().hmm_paged_attention_workspace_size(*sizes)


def rope_table(n_pos: int, rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """[n_pos, rotary_dim / 2, 2] fp32 (cos, sin) of p * theta^(-2i / rotary_dim), the
    angles in 64 bits: laid out once, for paged_kv_append."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * theta ** (-2.0 * i / rotary_dim)[None, :]
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous().to(device)


@_on_device
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
    dev, dtype, hk, d, cache = _cache(k_pages, v_pages)
    n_tokens = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else -1
    kp = _rows(k, "k", dtype, dev, (n_tokens, hk, d))
    vp = _rows(v, "v", dtype, dev, (n_tokens, hk, d))
    heads, qp, op = 0, (None, 0, 0), (None, 0, 0)
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must be [n_tokens, n_heads, D]")
        heads = q.shape[1]
        qp = _rows(q, "q", dtype, dev, (n_tokens, heads, d))
        if out is None:
            out = torch.empty((n_tokens, heads, d), dtype=dtype, device=q.device)
        op = _rows(out, "out", dtype, dev, (n_tokens, heads, d))
    batch = _batch(page_table, cu_new, kv_len, n_tokens, dev)
    wdt, wq, wk = -1, None, None
    if q_weight is not None or k_weight is not None:
        w = k_weight if q_weight is None else q_weight
        if not isinstance(w, torch.Tensor) or w.dtype not in (dtype, torch.float32):
            raise TypeError(f"norm weights must be float32 or {dtype}")
        wdt = HMM_DTYPE_F32 if w.dtype is torch.float32 else _DTYPES[dtype]
        if q_weight is not None:
            wq = _tensor(q_weight, "q_weight", w.dtype, dev, (d,))
        if k_weight is not None:
            wk = _tensor(k_weight, "k_weight", w.dtype, dev, (d,))
    rp, n_pos, rotary, pp = None, 0, 0, None
    if rope is not None:
        rp = _tensor(rope, "rope", torch.float32, dev)
        if rope.dim() != 3 or rope.shape[2] != 2:
            raise ValueError("rope must be [n_pos, pairs, 2]")
        n_pos, rotary = rope.shape[0], 2 * rope.shape[1]
    if positions is not None:
        pp = _tensor(positions, "positions", _i32, dev, (n_tokens,))
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_kv_append", C.byref(cache), C.byref(batch), qp[0], qp[1], qp[2], heads, kp[0],
         kp[1], kp[2], vp[0], vp[1], vp[2], wq, wk, wdt, eps, rp, n_pos, rotary, interleaved, pp, op[0],
         op[1], op[2], sp, stream)
    if waits:
        _wait(status, stream)
    return out


@_on_device
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
    dev, dtype, hk, d, cache = _cache(k_pages, v_pages)
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [n_tokens, n_heads, D]")
    n_tokens, heads, _ = shape = q.shape
    if shape[2] != d:
        raise ValueError(f"q has heads of {shape[2]}, the cache of {d}")
    qp, qt, qh = _rows(q, "q", dtype, dev, shape)
    batch = _batch(page_table, cu_new, kv_len, n_tokens, dev)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
    op = _tensor(out, "out", dtype, dev, shape)
    lse = torch.empty((n_tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    nws = _attention_workspace(dev, batch.n_seq, n_tokens, heads, hk, d)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device)
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_attention", C.byref(cache), C.byref(batch), qp, qt, qh, heads,
         d ** -0.5 if scale is None else scale, causal, window, sinks, max_new, op,
         lse.data_ptr() if return_lse else None, sp, ws.data_ptr(), nws, stream)
    if waits:
        _wait(status, stream)
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ pages


def _pages(t, name: str):
    """(pointer, n_layers, layer stride, n_pages, page stride, bytes of a page) in bytes, of
    [(n_layers,) n_pages, ...]; a page (all but the leading dimensions) must be one block."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    shape, strides, b = t.shape, t.stride(), t.element_size()
    lead = len(shape) == 5
    if not 3 <= len(shape) <= 5:
        raise ValueError(f"{name} must be [n_pages, n_kv_heads, page_tokens, D], with a leading "
                         "dimension of layers or not")
    need = 1
    for st, n in sorted(zip(strides[1 + lead:], shape[1 + lead:])):
        if n != 1:
            if st != need:
                raise ValueError(f"{name}: a page must be one block of memory")
            need *= n
    return (t.data_ptr(), shape[0] if lead else 1, strides[0] * b if lead else 0, shape[lead],
            strides[lead] * b, need * b)


def _store(k_pages, v_pages):
    """(device index, PageStore)."""
    kp, layers, kl, n, ks, size = _pages(k_pages, "k_pages")
    vp, _, vl, _, vs, _ = _pages(v_pages, "v_pages")
    dev = k_pages.get_device()
    if k_pages.shape != v_pages.shape or k_pages.dtype is not v_pages.dtype or v_pages.get_device() != dev:
        raise ValueError("k_pages and v_pages differ in shape, dtype or device")
    return dev, PageStore(kp, vp, n, size, layers, ks, kl, vs, vl)


def _state(page_table, refs, kv_len, out, dev):
    """(PagedState, [new page_table, refs, kv_len], workspace)."""
    tp, n_seq, pps = _table(page_table, dev)
    rp = _tensor(refs, "refs", _i32, dev)
    if refs.dim() != 1:
        raise ValueError("refs must be [n_pages]")
    n = refs.shape[0]
    old = [page_table, refs]
    lp = 0
    if kv_len is not None:
        lp = _tensor(kv_len, "kv_len", _i32, dev, (n_seq,))
        old.append(kv_len)
    if out is None:
        new = [torch.empty_like(t) for t in old]
        ptr = [t.data_ptr() for t in new]
    else:
        new = list(out)
        if len(new) != len(old):
            raise ValueError(f"out must hold {len(old)} tensors")
        ptr = [_tensor(t, f"out {name}", _i32, dev, o.shape)
               for t, o, name in zip(new, old, ("page_table", "refs", "kv_len"))]
    ws = torch.empty(_state_workspace(n_seq, n), dtype=torch.uint8, device=page_table.device)
    return PagedState(tp, rp, lp, ptr[0], ptr[1], ptr[2] if lp else 0, n_seq, pps, n), new, ws


@functools.lru_cache(maxsize=256)
def _state_workspace(n_seq: int, n_pages: int) -> int:
    return load().hmm_paged_state_workspace_size(n_seq, n_pages)


def _ids(t, name: str, dev: int, shape=None) -> int:
    p = _tensor(t, name, _i32, dev, shape)
    if t.dim() != 1:
        raise ValueError(f"{name} must be a vector")
    return p


def _device_of(t, name: str) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


@_on_device
def paged_copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor,
                     dst: torch.Tensor, *, status: torch.Tensor | None = None) -> None:
    """Copies page src[i] to page dst[i] (int32) of K and V, in every layer of
    [n_layers, n_pages, n_kv_heads, page_tokens, D] arrays; a pair with a negative entry
    is skipped.  Nothing is copied, and BOUNDS raised, if a page is out of range, a dst is
    listed twice or is another pair's src."""
    dev, store = _store(k_pages, v_pages)
    a = _ids(src, "src", dev)
    b = _ids(dst, "dst", dev, src.shape)
    ws = torch.empty(1, dtype=_i32, device=k_pages.device)
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_copy_pages", C.byref(store), a, b, src.shape[0], sp, ws.data_ptr(), 4, stream)
    if waits:
        _wait(status, stream)


@_on_device
def paged_free(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               seqs: torch.Tensor, *, out=None, status: torch.Tensor | None = None):
    """Frees the sequences of `seqs` (int32; one listed twice is freed once): their pages
    lose a reference each, their rows become -1 and their lengths 0.  Returns the new
    (page_table, refs, kv_len): new tensors, or `out`, which may be the old ones."""
    dev = _device_of(page_table, "page_table")
    state, new, ws = _state(page_table, refs, kv_len, out, dev)
    a = _ids(seqs, "seqs", dev)
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_free", C.byref(state), a, seqs.shape[0], sp, ws.data_ptr(), ws.numel(), stream)
    if waits:
        _wait(status, stream)
    return tuple(new)


@_on_device
def paged_fork(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               src: torch.Tensor, dst: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               *, out=None, status: torch.Tensor | None = None):
    """Forks sequence src[i] into the empty row dst[i]: full pages are shared, a partly
    filled last page is copied into the lowest free one (in every layer of
    [n_layers, n_pages, ...] arrays).  Returns the new (page_table, refs, kv_len) as
    paged_free does.  A request that cannot be met as a whole changes nothing."""
    dev, store = _store(k_pages, v_pages)
    state, new, ws = _state(page_table, refs, kv_len, out, dev)
    a = _ids(src, "src", dev)
    b = _ids(dst, "dst", dev, src.shape)
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_fork", C.byref(state), C.byref(store), k_pages.shape[-2], a, b, src.shape[0], sp,
         ws.data_ptr(), ws.numel(), stream)
    if waits:
        _wait(status, stream)
    return tuple(new)


@_on_device
def paged_grow(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               n_new: torch.Tensor, page_tokens: int, *, out=None,
               status: torch.Tensor | None = None):
    """Makes room for n_new[s] more tokens of every sequence: entries of the pages they
    touch that hold none get the lowest free pages, in row order.  Returns the new
    (page_table, refs, kv_len + n_new) as paged_free does."""
    dev = _device_of(page_table, "page_table")
    state, new, ws = _state(page_table, refs, kv_len, out, dev)
    a = _ids(n_new, "n_new", dev, kv_len.shape)
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_grow", C.byref(state), page_tokens, a, sp, ws.data_ptr(), ws.numel(), stream)
    if waits:
        _wait(status, stream)
    return tuple(new)


@_on_device
def paged_compact(page_table: torch.Tensor, refs: torch.Tensor, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, *, out=None, status: torch.Tensor | None = None):
    """Moves the live pages (refs != 0) to the front of the cache, each at most once: the
    k-th live page behind the front goes to the k-th free one in it.  Returns
    (page_table, refs, live [1] int32); `out` holds the first two.  Page numbers kept
    elsewhere than in page_table do not follow."""
    dev, store = _store(k_pages, v_pages)
    state, new, ws = _state(page_table, refs, None, out, dev)
    live = torch.empty(1, dtype=_i32, device=k_pages.device)
    status, sp, waits = _status(status, dev)
    stream = _raw_stream(dev)
    call("hmm_paged_compact", C.byref(state), C.byref(store), live.data_ptr(), sp, ws.data_ptr(),
         ws.numel(), stream)
    if waits:
        _wait(status, stream)
    return (*new, live)

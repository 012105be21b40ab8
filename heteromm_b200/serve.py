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
import importlib.util
import threading

import torch

from . import build as _build
from ._abi import HmmError, last_error, load

# What these calls do with their arguments is in src/py/serve_calls.cpp: they are issued
# once per layer and token, where checks in Python take longer than the kernels.
_ENTRIES = ("hmm_paged_kv_append", "hmm_paged_attention", "hmm_paged_attention_workspace_size",
            "hmm_paged_state_workspace_size", "hmm_paged_copy_pages", "hmm_paged_free", "hmm_paged_fork",
            "hmm_paged_grow", "hmm_paged_compact", "hmm_status_read")


def _raise(name: str, status: int):
    raise HmmError(status, name, last_error())


class _Calls:
    """The module heteromm_serve_calls, loaded (and built, if it is absent) at the first call."""

    _lock = threading.Lock()

    def __getattr__(self, name: str):
        if name not in ("attention", "append", "copy_pages", "free", "fork", "grow", "compact"):
            raise AttributeError(name)
        with self._lock:
            if name not in self.__dict__:     # (another thread's first call was quicker)
                path = _build.build_serve_calls()
                if not path:
                    raise RuntimeError("the serving calls need torch's headers and its CUDA library to be built")
                spec = importlib.util.spec_from_file_location("heteromm_serve_calls", path)
                native = importlib.util.module_from_spec(spec)
                lib = load()
                native.bind(*(C.cast(getattr(lib, e), C.c_void_p).value for e in _ENTRIES), _raise)
                for f in ("attention", "append", "copy_pages", "free", "fork", "grow", "compact"):
                    setattr(self, f, getattr(native, f))
        return self.__dict__[name]


_calls = _Calls()


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
    keys and values into the cache.  Returns the queries (in `out`, which may be q, or rows
    that overlap neither q nor k nor v).

    q [n_tokens, n_heads, D] (or None: keys and values alone), k, v
    [n_tokens, n_kv_heads, D], views of one projection included.  Pairs are halves
    (i, i + pairs), or neighbours with `interleaved`; the angle's row is the token's
    position, or positions [n_tokens] int32."""
    return _calls.append(q, k, v, k_pages, v_pages, page_table, cu_new, kv_len, rope, q_weight, k_weight, eps,
                         interleaved, positions, out, status)


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
    return _calls.attention(q, k_pages, v_pages, page_table, cu_new, kv_len, causal, window, sinks, scale, max_new,
                            return_lse, out, status)


# ------------------------------------------------------------------ pages


def paged_copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor,
                     dst: torch.Tensor, *, status: torch.Tensor | None = None) -> None:
    """Copies page src[i] to page dst[i] (int32) of K and V, in every layer of
    [n_layers, n_pages, n_kv_heads, page_tokens, D] arrays; a pair with a negative entry
    is skipped.  Nothing is copied, and BOUNDS raised, if a page is out of range, a dst is
    listed twice or is another pair's src."""
    return _calls.copy_pages(k_pages, v_pages, src, dst, status)


def paged_free(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               seqs: torch.Tensor, *, out=None, status: torch.Tensor | None = None):
    """Frees the sequences of `seqs` (int32; one listed twice is freed once): their pages
    lose a reference each, their rows become -1 and their lengths 0.  Returns the new
    (page_table, refs, kv_len): new tensors, or `out`, each of which may be the old one
    itself (or is apart from all that the call reads)."""
    return _calls.free(page_table, refs, kv_len, seqs, out, status)


def paged_fork(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               src: torch.Tensor, dst: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               *, out=None, status: torch.Tensor | None = None):
    """Forks sequence src[i] into the empty row dst[i]: full pages are shared, a partly
    filled last page is copied into the lowest free one (in every layer of
    [n_layers, n_pages, ...] arrays).  Returns the new (page_table, refs, kv_len) as
    paged_free does.  A request that cannot be met as a whole changes nothing."""
    return _calls.fork(page_table, refs, kv_len, src, dst, k_pages, v_pages, out, status)


def paged_grow(page_table: torch.Tensor, refs: torch.Tensor, kv_len: torch.Tensor,
               n_new: torch.Tensor, page_tokens: int, *, out=None,
               status: torch.Tensor | None = None):
    """Makes room for n_new[s] more tokens of every sequence: entries of the pages they
    touch that hold none get the lowest free pages, in row order.  Returns the new
    (page_table, refs, kv_len + n_new) as paged_free does."""
    return _calls.grow(page_table, refs, kv_len, n_new, page_tokens, out, status)


def paged_compact(page_table: torch.Tensor, refs: torch.Tensor, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, *, out=None, status: torch.Tensor | None = None):
    """Moves the live pages (refs != 0) to the front of the cache, each at most once: the
    k-th live page behind the front goes to the k-th free one in it.  Returns
    (page_table, refs, live [1] int32); `out` holds the first two.  Page numbers kept
    elsewhere than in page_table do not follow."""
    return _calls.compact(page_table, refs, k_pages, v_pages, out, status)

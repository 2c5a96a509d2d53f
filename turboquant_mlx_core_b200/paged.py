"""The paged 8-bit KV cache of a server's requests (include/turboquant_c/turboquant_b200.h, tq_paged_*).

The reference's cache holds one sequence (include/turboquant/kv_cache.h:42-133; TQKVCache here); this one holds many, in pages, with
their lengths on the device.  A step:

    cache.plan(counts, tokens, max_count, positions=positions)     # tables, slots and positions of the new tokens
    for each layer:
        ...                                                        # projections; rotary embedding by `positions`
        cache.append(layer, k, v)
        cache.attention(layer, q, out=out)

Tensors are torch CUDA tensors; rows, counts and lengths may be int32 numpy arrays, counts and lengths any whole numbers that fit.  Everything runs in the
CUDA library.
"""
from __future__ import annotations

import numpy as np

from . import _lib
from ._lib import TQ_F16, TQ_F32, TQError, check
from .api import _stream_ptr

# A decode step's calls move microseconds of work each: their Python side is a handful of look-ups, and types are told by identity.
_torch = None


def _load_torch():
    global _torch
    if _torch is None:
        import torch
        _torch = torch
    return _torch


def _fits(n, what):
    """(The C interface takes the low 32 bits of any number.)"""
    if -0x80000000 <= n <= 0x7fffffff:
        return n
    raise ValueError(f"{what} must fit in 32 bits, got {n}")


def _host_ints(x, what):
    """Whole numbers in host memory, of any integer type, as contiguous int32."""
    x = np.asarray(x)
    if x.dtype != np.int32 and x.size:
        if x.dtype.kind not in "iu":
            raise TypeError(f"{what} must be whole numbers, got {x.dtype}")
        _fits(int(x.min()), what)
        _fits(int(x.max()), what)
    return np.ascontiguousarray(x, np.int32)


def _ints(x, what, n):
    """Address of n whole numbers of 32 bits, contiguous."""
    if x is None:
        return None
    if hasattr(x, "data_ptr"):
        fine, contiguous, size, at = x.dtype is _torch.int32, x.is_contiguous(), x.numel(), x.data_ptr()
    else:
        fine, contiguous, size, at = x.dtype == np.int32, x.flags["C_CONTIGUOUS"], x.size, x.ctypes.data
    if not fine:
        raise TypeError(f"{what} must be int32, got {x.dtype}")
    if not contiguous:
        raise ValueError(f"{what} must be contiguous")
    if size != n:
        raise ValueError(f"{what} must have {n} elements")
    return at


def _rows(x, heads, dim, what):
    """[tokens, heads, dim] with contiguous heads (`heads` 0: any number of them): address, tokens, heads, elements from token to token."""
    if not hasattr(x, "data_ptr"):
        raise TypeError(f"{what} must be a torch CUDA tensor")
    try:
        tokens, n, d = x.shape
        step, head, one = x.stride()
    except ValueError:
        d = None
    if d != dim or (heads and n != heads):
        raise ValueError(f"{what} must be [tokens, {heads or 'heads'}, {dim}]")
    if one != 1 or (head != dim and n > 1):
        raise ValueError(f"the heads of a token of {what} must be contiguous")
    return x.data_ptr(), tokens, n, step if tokens > 1 else max(n * dim, step)


def _tag(x, what):
    if x.dtype is _torch.float16:
        return TQ_F16
    if x.dtype is _torch.float32:
        return TQ_F32
    raise TypeError(f"{what}: expected float32 or float16, got {x.dtype}")


def _zeros_like(x, stream):
    """Zeros in front of a call on `stream`, by that stream."""
    if not x.is_cuda:
        return x.new_zeros(x.shape)
    cuda = _torch.cuda
    if stream is None:
        stream = cuda.default_stream(x.device)
    elif not hasattr(stream, "cuda_stream"):
        stream = cuda.ExternalStream(int(stream), x.device)
    with cuda.stream(stream):
        return x.new_zeros(x.shape)


class PagedKVCache:
    """Keys and values of up to `max_requests` requests in `num_pages` pages of `page_tokens` tokens, 8 bits each with a power of
    two for each page and head."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, num_pages: int, page_tokens: int = 64, max_requests: int = 256,
                 max_pages_per_request: int | None = None, max_tokens: int = 8192):
        self._L = _lib.load()
        self.num_layers, self.num_heads, self.head_dim = _fits(int(num_layers), "num_layers"), _fits(int(num_heads), "num_heads"), _fits(int(head_dim), "head_dim")
        self.num_pages, self.page_tokens = _fits(int(num_pages), "num_pages"), _fits(int(page_tokens), "page_tokens")
        self.max_requests, self.max_tokens = _fits(int(max_requests), "max_requests"), _fits(int(max_tokens), "max_tokens")
        self.max_pages_per_request = self.num_pages if max_pages_per_request is None else _fits(int(max_pages_per_request), "max_pages_per_request")
        self._h = self._L.tq_paged_cache_create(self.num_layers, self.num_heads, self.head_dim, self.num_pages, self.page_tokens,
                                                self.max_requests, self.max_pages_per_request, self.max_tokens)
        if not self._h:
            raise TQError("PagedKVCache: " + _lib.last_error())
        _load_torch()

    @property
    def handle(self):
        return self._h

    def plan(self, counts, tokens: int | None = None, max_count: int | None = None, rows=None, starts=None, lengths=None, slots=None,
             positions=None, tables=None, stream=None):
        """counts[i] new tokens for the request in row rows[i] (row i without rows).  `tokens` and `max_count`: the most that there can be in
        all and for one request (taken from counts where that is in host memory: a numpy array or a list).  starts [n + 1], lengths [n], slots [tokens],
        positions [tokens] and tables [n, width]: int32 tensors that are filled, each of them optional."""
        if not hasattr(counts, "data_ptr"):
            counts = _host_ints(counts, "counts")
            tokens = int(counts.sum()) if tokens is None else tokens
            max_count = int(counts.max(initial=0)) if max_count is None else max_count
        elif tokens is None or max_count is None:
            raise ValueError("plan: counts on the device need tokens and max_count")
        n, width = counts.shape[0], 0
        _fits(tokens, "tokens")
        _fits(max_count, "max_count")
        if tables is not None:
            if len(tables.shape) != 2 or tables.shape[0] != n:
                raise ValueError("plan: tables must be [n, width]")
            width = tables.shape[1]
        if self._L.tq_paged_plan(self._h, _ints(rows, "rows", n), _ints(counts, "counts", n), n, tokens, max_count, _ints(starts, "starts", n + 1),
                                 _ints(lengths, "lengths", n), _ints(slots, "slots", tokens), _ints(positions, "positions", tokens),
                                 _ints(tables, "tables", n * width), width, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.plan")

    def truncate(self, lengths, rows=None, stream=None):
        """The request in row rows[i] (row i without rows) keeps its first lengths[i] tokens; 0 releases it."""
        if not hasattr(lengths, "data_ptr"):
            lengths = _host_ints(lengths, "lengths")
        n = lengths.shape[0]
        if self._L.tq_paged_truncate(self._h, _ints(rows, "rows", n), _ints(lengths, "lengths", n), n, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.truncate")

    def append(self, layer: int, keys, values, stream=None):
        """Keys and values of the planned tokens, [tokens, heads, head_dim] fp32 or fp16; a token's heads are contiguous, tokens may be apart."""
        kp, tokens, _, ks = _rows(keys, self.num_heads, self.head_dim, "keys")
        vp, more, _, vs = _rows(values, self.num_heads, self.head_dim, "values")
        if tokens != more or keys.dtype is not values.dtype:
            raise ValueError("keys and values must have the same number of tokens and type")
        if self._L.tq_paged_append(self._h, _fits(layer, "layer"), kp, vp, _tag(keys, "append"), tokens, ks, vs, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.append")

    def attention(self, layer: int, queries, window: int = 0, scale: float = 0.0, out=None, lse=None, stream=None):
        """Causal attention of the planned tokens' queries, fp16 [tokens, q_heads, head_dim], over their requests; returns out.  A `window` of w
        lets a token see itself and the w - 1 before it.  lse: fp32 [tokens, q_heads], filled with the log of the softmax denominators."""
        qp, tokens, q_heads, qs = _rows(queries, 0, self.head_dim, "queries")
        half = _torch.float16
        if queries.dtype is not half:
            raise TypeError("attention: queries must be float16")
        if out is None:
            out = _zeros_like(queries, stream)
        op, more, _, os_ = _rows(out, q_heads, self.head_dim, "out")
        if more != tokens or out.dtype is not half:
            raise ValueError("out must be float16 of the queries' shape")
        lp = None
        if lse is not None:
            if lse.dtype is not _torch.float32 or lse.shape != (tokens, q_heads) or not lse.is_contiguous():
                raise ValueError("lse must be contiguous float32 [tokens, q_heads]")
            lp = lse.data_ptr()
        if self._L.tq_paged_attention(self._h, _fits(layer, "layer"), qp, tokens, q_heads, qs, _fits(window, "window"), scale, op, os_, lp, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.attention")
        return out

    def read_pages(self, layer: int, pages, keys=None, values=None, stream=None):
        """The values that whole pages hold (their numbers: an int32 tensor), into keys and values, [n, page_tokens, heads, head_dim] fp32 or
        fp16 tensors, either of them None."""
        n, tag, at = pages.shape[0], None, [None, None]
        for i, x in enumerate((keys, values)):
            if x is None:
                continue
            if x.shape != (n, self.page_tokens, self.num_heads, self.head_dim) or not x.is_contiguous():
                raise ValueError(f"keys and values must be contiguous {[n, self.page_tokens, self.num_heads, self.head_dim]}")
            if tag not in (None, _tag(x, "read_pages")):
                raise ValueError("keys and values must have the same type")
            tag, at[i] = _tag(x, "read_pages"), x.data_ptr()
        if self._L.tq_paged_read(self._h, _fits(layer, "layer"), _ints(pages, "pages", n), n, *at, TQ_F16 if tag is None else tag,
                                 None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.read_pages")

    def free_pages(self) -> int:
        """Free pages, once all work is done (waits for the device)."""
        n = self._L.tq_paged_free_pages(self._h)
        if n < 0:
            check(-1, "PagedKVCache.free_pages")
        return n

    def check_status(self):
        """Raise if a finished call found its batch impossible or another plan on the device than its own (then nothing of it was done), or a wait on the
        device ran out."""
        check(self._L.tq_paged_status(self._h), "PagedKVCache")

    def close(self):
        if getattr(self, "_h", None):
            self._L.tq_paged_cache_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

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
_torch = _int32 = _float16 = _float32 = None


def _load_torch():
    global _torch, _int32, _float16, _float32
    if _torch is None:
        import torch
        _torch, _int32, _float16, _float32 = torch, torch.int32, torch.float16, torch.float32
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


def _elsewhere(x, device, what):
    """A tensor that is not on the cache's device: in host memory (the C interface takes or refuses it) or on another one."""
    if x.get_device() >= 0:
        raise ValueError(f"{what} is on cuda:{x.get_device()}, the cache on cuda:{device}")


def _ints(x, what, n, device):
    """Address of n whole numbers of 32 bits, contiguous."""
    if x is None:
        return None
    its = getattr(x, "get_device", None)
    if its is not None:
        if its() != device:
            _elsewhere(x, device, what)
        fine, contiguous, size, at = x.dtype is _int32, x.is_contiguous(), x.numel(), x.data_ptr()
    else:
        fine, contiguous, size, at = x.dtype == np.int32, x.flags["C_CONTIGUOUS"], x.size, x.ctypes.data
    if not fine:
        raise TypeError(f"{what} must be int32, got {x.dtype}")
    if not contiguous:
        raise ValueError(f"{what} must be contiguous")
    if size != n:
        raise ValueError(f"{what} must have {n} elements")
    return at


def _rows(x, heads, dim, what, device):
    """[tokens, heads, dim] with contiguous heads (`heads` 0: any number of them): address, tokens, heads, elements from token to token."""
    its = getattr(x, "get_device", None)
    if its is None:
        raise TypeError(f"{what} must be a torch CUDA tensor")
    if its() != device:
        _elsewhere(x, device, what)
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
    if x.dtype is _float16:
        return TQ_F16
    if x.dtype is _float32:
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
    two for each page and head, on the device that is current here."""

    _device = -1       # no CUDA device's number

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
        self._device = _load_torch().cuda.current_device()

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
        if not 0 <= tokens <= 0x7fffffff or not 0 <= max_count <= 0x7fffffff:
            _fits(tokens, "tokens")
            _fits(max_count, "max_count")
        if tables is not None:
            if len(tables.shape) != 2 or tables.shape[0] != n:
                raise ValueError("plan: tables must be [n, width]")
            width = tables.shape[1]
        on = self._device
        if self._L.tq_paged_plan(self._h, _ints(rows, "rows", n, on), _ints(counts, "counts", n, on), n, tokens, max_count, _ints(starts, "starts", n + 1, on),
                                 _ints(lengths, "lengths", n, on), _ints(slots, "slots", tokens, on), _ints(positions, "positions", tokens, on),
                                 _ints(tables, "tables", n * width, on), width, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.plan")

    def truncate(self, lengths, rows=None, stream=None):
        """The request in row rows[i] (row i without rows) keeps its first lengths[i] tokens; 0 releases it."""
        if not hasattr(lengths, "data_ptr"):
            lengths = _host_ints(lengths, "lengths")
        n = lengths.shape[0]
        on = self._device
        if self._L.tq_paged_truncate(self._h, _ints(rows, "rows", n, on), _ints(lengths, "lengths", n, on), n, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.truncate")

    def append(self, layer: int, keys, values, stream=None):
        """Keys and values of the planned tokens, [tokens, heads, head_dim] fp32 or fp16; a token's heads are contiguous, tokens may be apart."""
        kp, tokens, _, ks = _rows(keys, self.num_heads, self.head_dim, "keys", self._device)
        vp, more, _, vs = _rows(values, self.num_heads, self.head_dim, "values", self._device)
        if tokens != more or keys.dtype is not values.dtype:
            raise ValueError("keys and values must have the same number of tokens and type")
        if not 0 <= layer <= 0x7fffffff:
            _fits(layer, "layer")
        if self._L.tq_paged_append(self._h, layer, kp, vp, _tag(keys, "append"), tokens, ks, vs, None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.append")

    def attention(self, layer: int, queries, window: int = 0, scale: float = 0.0, out=None, lse=None, stream=None):
        """Causal attention of the planned tokens' queries, fp16 [tokens, q_heads, head_dim], over their requests; returns out.  A `window` of w
        lets a token see itself and the w - 1 before it.  lse: fp32 [tokens, q_heads], filled with the log of the softmax denominators."""
        qp, tokens, q_heads, qs = _rows(queries, 0, self.head_dim, "queries", self._device)
        if queries.dtype is not _float16:
            raise TypeError("attention: queries must be float16")
        if out is None:
            out = _zeros_like(queries, stream)
        op, more, _, os_ = _rows(out, q_heads, self.head_dim, "out", self._device)
        if more != tokens or out.dtype is not _float16:
            raise ValueError("out must be float16 of the queries' shape")
        lp = None
        if lse is not None:
            if lse.dtype is not _float32 or lse.shape != (tokens, q_heads) or not lse.is_contiguous():
                raise ValueError("lse must be contiguous float32 [tokens, q_heads]")
            if lse.get_device() != self._device:
                _elsewhere(lse, self._device, "lse")
            lp = lse.data_ptr()
        if not 0 <= layer <= 0x7fffffff or not 0 <= window <= 0x7fffffff:
            _fits(layer, "layer")
            _fits(window, "window")
        if self._L.tq_paged_attention(self._h, layer, qp, tokens, q_heads, qs, window, scale, op, os_, lp, None if stream is None else _stream_ptr(stream)):
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
            if x.get_device() != self._device:
                _elsewhere(x, self._device, "keys and values")
            tag, at[i] = _tag(x, "read_pages"), x.data_ptr()
        if self._L.tq_paged_read(self._h, _fits(layer, "layer"), _ints(pages, "pages", n, self._device), n, *at, TQ_F16 if tag is None else tag,
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

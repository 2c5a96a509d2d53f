"""The paged 8-bit KV cache of a server's requests (include/turboquant_c/turboquant_b200.h, tq_paged_*).

The reference's cache holds one sequence (include/turboquant/kv_cache.h:42-133; TQKVCache here); this one holds many, in pages, with
their lengths on the device.  A step:

    cache.plan(counts, tokens, max_count, positions=positions)     # tables, slots and positions of the new tokens
    for each layer:
        ...                                                        # projections; rotary embedding by `positions`
        cache.append(layer, k, v)
        cache.attention(layer, q, out=out)

Tensors are torch CUDA tensors; rows, counts and lengths may be int32 numpy arrays.  Everything runs in the CUDA library.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import TQ_F16, TQ_F32, TQError, check
from .api import _stream_ptr


def _ints(x, what, n=None):
    """Address of whole numbers of 32 bits, contiguous; `n`: how many there must be."""
    if x is None:
        return None
    tensor = hasattr(x, "data_ptr")
    if str(x.dtype).rpartition(".")[2] != "int32":
        raise TypeError(f"{what} must be int32, got {x.dtype}")
    if not (x.is_contiguous() if tensor else x.flags["C_CONTIGUOUS"]):
        raise ValueError(f"{what} must be contiguous")
    if n is not None and (x.numel() if tensor else x.size) != n:
        raise ValueError(f"{what} must have {n} elements")
    return x.data_ptr() if tensor else x.ctypes.data


def _rows(x, heads, dim, what):
    """[tokens, heads, dim] with contiguous heads: address, tokens, elements from token to token."""
    if not hasattr(x, "data_ptr"):
        raise TypeError(f"{what} must be a torch CUDA tensor")
    if len(x.shape) != 3 or (heads and x.shape[1] != heads) or x.shape[2] != dim:
        raise ValueError(f"{what} must be [tokens, {heads or 'heads'}, {dim}]")
    stride = x.stride()
    if stride[2] != 1 or (x.shape[1] > 1 and stride[1] != dim):
        raise ValueError(f"the heads of a token of {what} must be contiguous")
    row = x.shape[1] * dim
    return x.data_ptr(), x.shape[0], stride[0] if x.shape[0] > 1 else max(row, stride[0])


def _tag(x, what):
    name = str(x.dtype)
    if name.endswith("float16") and "bfloat" not in name:
        return TQ_F16
    if name.endswith("float32"):
        return TQ_F32
    raise TypeError(f"{what}: expected float32 or float16, got {x.dtype}")


class PagedKVCache:
    """Keys and values of up to `max_requests` requests in `num_pages` pages of `page_tokens` tokens, 8 bits each with a power of
    two for each page and head."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, num_pages: int, page_tokens: int = 64, max_requests: int = 256,
                 max_pages_per_request: int | None = None, max_tokens: int = 8192):
        self._L = _lib.load()
        self.num_layers, self.num_heads, self.head_dim = int(num_layers), int(num_heads), int(head_dim)
        self.num_pages, self.page_tokens, self.max_requests = int(num_pages), int(page_tokens), int(max_requests)
        self.max_pages_per_request = self.num_pages if max_pages_per_request is None else int(max_pages_per_request)
        self.max_tokens = int(max_tokens)
        self._h = self._L.tq_paged_cache_create(self.num_layers, self.num_heads, self.head_dim, self.num_pages, self.page_tokens,
                                                self.max_requests, self.max_pages_per_request, self.max_tokens)
        if not self._h:
            raise TQError("PagedKVCache: " + _lib.last_error())

    @property
    def handle(self):
        return self._h

    def plan(self, counts, tokens: int | None = None, max_count: int | None = None, rows=None, starts=None, lengths=None, slots=None,
             positions=None, tables=None, stream=None):
        """counts[i] new tokens for the request in row rows[i] (row i without rows).  `tokens` and `max_count`: the most that there can be in
        all and for one request (taken from counts where that is a numpy array).  starts [n + 1], lengths [n], slots [tokens],
        positions [tokens] and tables [n, width]: int32 tensors that are filled, each of them optional."""
        if not hasattr(counts, "data_ptr"):
            counts = np.ascontiguousarray(counts, np.int32)
            tokens = int(counts.sum()) if tokens is None else tokens
            max_count = int(counts.max(initial=0)) if max_count is None else max_count
        elif tokens is None or max_count is None:
            raise ValueError("plan: counts on the device need tokens and max_count")
        n = int(counts.shape[0])
        if tables is not None and (len(tables.shape) != 2 or tables.shape[0] != n):
            raise ValueError("plan: tables must be [n, width]")
        check(self._L.tq_paged_plan(self._h, _ints(rows, "rows", n), _ints(counts, "counts", n), n, int(tokens), int(max_count),
                                    _ints(starts, "starts", n + 1), _ints(lengths, "lengths", n), _ints(slots, "slots", tokens),
                                    _ints(positions, "positions", tokens), _ints(tables, "tables"),
                                    0 if tables is None else int(tables.shape[1]), _stream_ptr(stream)), "PagedKVCache.plan")

    def truncate(self, lengths, rows=None, stream=None):
        """The request in row rows[i] (row i without rows) keeps its first lengths[i] tokens; 0 releases it."""
        if not hasattr(lengths, "data_ptr"):
            lengths = np.ascontiguousarray(lengths, np.int32)
        n = int(lengths.shape[0])
        check(self._L.tq_paged_truncate(self._h, _ints(rows, "rows", n), _ints(lengths, "lengths", n), n, _stream_ptr(stream)),
              "PagedKVCache.truncate")

    def append(self, layer: int, keys, values, stream=None):
        """Keys and values of the planned tokens, [tokens, heads, head_dim] fp32 or fp16; a token's heads are contiguous, tokens may be apart."""
        kp, tokens, ks = _rows(keys, self.num_heads, self.head_dim, "keys")
        vp, more, vs = _rows(values, self.num_heads, self.head_dim, "values")
        if tokens != more or keys.dtype != values.dtype:
            raise ValueError("keys and values must have the same number of tokens and type")
        check(self._L.tq_paged_append(self._h, int(layer), kp, vp, _tag(keys, "append"), tokens, ks, vs, _stream_ptr(stream)),
              "PagedKVCache.append")

    def attention(self, layer: int, queries, window: int = 0, scale: float = 0.0, out=None, lse=None, stream=None):
        """Causal attention of the planned tokens' queries, fp16 [tokens, q_heads, head_dim], over their requests; returns out.  A `window` of w
        lets a token see itself and the w - 1 before it.  lse: fp32 [tokens, q_heads], filled with the log of the softmax denominators."""
        qp, tokens, qs = _rows(queries, None, self.head_dim, "queries")
        if _tag(queries, "attention") != TQ_F16:
            raise TypeError("attention: queries must be float16")
        if out is None:
            out = queries.new_zeros(queries.shape)
        op, more, os_ = _rows(out, int(queries.shape[1]), self.head_dim, "out")
        if more != tokens or _tag(out, "attention") != TQ_F16:
            raise ValueError("out must be float16 of the queries' shape")
        if lse is not None and (tuple(lse.shape) != tuple(queries.shape[:2]) or _tag(lse, "attention") != TQ_F32 or not lse.is_contiguous()):
            raise ValueError("lse must be contiguous float32 [tokens, q_heads]")
        check(self._L.tq_paged_attention(self._h, int(layer), qp, tokens, int(queries.shape[1]), qs, int(window), float(scale), op, os_,
                                         None if lse is None else lse.data_ptr(), _stream_ptr(stream)), "PagedKVCache.attention")
        return out

    def read_pages(self, layer: int, pages, keys=None, values=None, stream=None):
        """The values that whole pages hold (their numbers: an int32 tensor), into keys and values, [n, page_tokens, heads, head_dim] fp32 or
        fp16 tensors, either of them None."""
        n = int(pages.shape[0])
        shape, tags = (n, self.page_tokens, self.num_heads, self.head_dim), set()
        for x in (keys, values):
            if x is None:
                continue
            if tuple(x.shape) != shape or not x.is_contiguous():
                raise ValueError(f"keys and values must be contiguous {list(shape)}")
            tags.add(_tag(x, "read_pages"))
        if len(tags) > 1:
            raise ValueError("keys and values must have the same type")
        check(self._L.tq_paged_read(self._h, int(layer), _ints(pages, "pages", n), n, None if keys is None else keys.data_ptr(),
                                    None if values is None else values.data_ptr(), tags.pop() if tags else TQ_F16, _stream_ptr(stream)),
              "PagedKVCache.read_pages")

    def free_pages(self) -> int:
        """Free pages, once all work is done (waits for the device)."""
        n = self._L.tq_paged_free_pages(self._h)
        if n < 0:
            check(-1, "PagedKVCache.free_pages")
        return n

    def check_status(self):
        """Raise if a finished call found its batch impossible (then nothing of the batch was done) or a wait on the device ran out."""
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

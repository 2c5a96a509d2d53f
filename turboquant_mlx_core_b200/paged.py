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
    if (tokens | n | d) > 0x7fffffff:
        raise ValueError(f"the sizes of {what} must fit in 32 bits")
    if one != 1 or (head != dim and n > 1):
        raise ValueError(f"the heads of a token of {what} must be contiguous")
    return x.data_ptr(), tokens, n, step if tokens > 1 else max(n * dim, step)


def _number(x, what):
    if len(x.shape) != 1:
        raise ValueError(f"{what} must have one dimension")
    return _fits(x.shape[0], f"the size of {what}")


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
    _planned = 0       # tokens of the last plan

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
        self._planned = tokens

    def tree(self, parents=None, positions=None, stream=None):
        """The planned tokens are trees of drafts: parents, an int32 tensor [tokens], is each token's parent, counted from its request's first new
        token and in front of it, or -1; None: chains.  positions: int32 [tokens], filled with what a request held before and the token's depth."""
        if parents is None and positions is None:
            tokens = self._planned
        else:
            tokens = _number(parents if parents is not None else positions, "parents and positions")
        if self._L.tq_paged_tree(self._h, _ints(parents, "parents", tokens, self._device), tokens, _ints(positions, "positions", tokens, self._device),
                                 None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.tree")

    def keep(self, path, kept, lengths=None, stream=None):
        """Of each request's new tokens kept[i] stay, those that path[i] lists in ascending order (all of them where kept[i] is below 0), as
        `verify_drafts` gives them; they move up in all layers, and the pages behind become free.  path [n, width], kept [n] and lengths [n] (filled with
        the tokens that each request holds then) are int32 tensors."""
        if len(path.shape) != 2:
            raise ValueError("keep: path must be [n, width]")
        n, width = path.shape
        if (n | width) > 0x7fffffff:
            raise ValueError("the sizes of path must fit in 32 bits")
        on = self._device
        if self._L.tq_paged_keep(self._h, _ints(path, "path", n * width, on), width, _ints(kept, "kept", n, on), n, _ints(lengths, "lengths", n, on),
                                 None if stream is None else _stream_ptr(stream)):
            check(-1, "PagedKVCache.keep")

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
        return self._attend(self._L.tq_paged_attention, "attention", layer, queries, window, scale, out, lse, stream)

    def tree_attention(self, layer: int, queries, window: int = 0, scale: float = 0.0, out=None, lse=None, stream=None):
        """The same for tokens that are trees of drafts (`tree`): a token sees those in front of its request's new ones, its ancestors and itself.
        Where all are chains `attention` gives the same, faster for few rows of a request and for prompts."""
        return self._attend(self._L.tq_paged_tree_attention, "tree_attention", layer, queries, window, scale, out, lse, stream)

    def _attend(self, call, name, layer, queries, window, scale, out, lse, stream):
        qp, tokens, q_heads, qs = _rows(queries, 0, self.head_dim, "queries", self._device)
        if queries.dtype is not _float16:
            raise TypeError(f"{name}: queries must be float16")
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
        if call(self._h, layer, qp, tokens, q_heads, qs, window, scale, op, os_, lp, None if stream is None else _stream_ptr(stream)):
            check(-1, f"PagedKVCache.{name}")
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


def _device_of(x, what):
    its = getattr(x, "get_device", None)
    if its is None:
        raise TypeError(f"{what} must be a torch CUDA tensor")
    return its()


def qk_norm_rope(queries, keys, query_weight, key_weight, positions, theta: float = 10000.0, eps: float = 1e-6, out=None, stream=None):
    """The norm of each head of queries and keys, fp16 [tokens, heads, head_dim], and its rotation by `positions` (int32 [tokens]; what `plan` and `tree`
    give) in one pass; a token's heads are contiguous, tokens may be apart.  The weights are fp16 [head_dim].  out: a pair of tensors that share no
    memory with the arguments, None: in place.  Returns the pair."""
    _load_torch()
    on = _device_of(queries, "queries")
    if len(queries.shape) != 3:
        raise ValueError("queries must be [tokens, heads, head_dim]")
    dim = queries.shape[2]
    qp, tokens, q_heads, qs = _rows(queries, 0, dim, "queries", on)
    kp, more, kv_heads, ks = _rows(keys, 0, dim, "keys", on)
    if out is None:
        out, qo, qt, ko, kt, qn, kn = (queries, keys), qp, qs, kp, ks, tokens, tokens
    else:
        qo, qn, _, qt = _rows(out[0], q_heads, dim, "out", on)
        ko, kn, _, kt = _rows(out[1], kv_heads, dim, "out", on)
    if not tokens == more == qn == kn:
        raise ValueError("queries, keys and out must have the same number of tokens")
    half = _float16
    if not (queries.dtype is half and keys.dtype is half and out[0].dtype is half and out[1].dtype is half and query_weight.dtype is half and key_weight.dtype is half):
        raise TypeError("queries, keys, weights and out must be float16")
    for w in (query_weight, key_weight):
        if w.shape != (dim,) or not w.is_contiguous():
            raise ValueError(f"weights must be contiguous, [{dim}]")
        if w.get_device() != on:
            raise ValueError("weights are on another device than the queries")
    if _lib.load().tq_qk_norm_rope_f16(qp, kp, query_weight.data_ptr(), key_weight.data_ptr(), _ints(positions, "positions", tokens, on), tokens, q_heads, kv_heads, dim,
                                       qs, ks, eps, theta, qo, ko, qt, kt, None if stream is None else _stream_ptr(stream)):
        check(-1, "qk_norm_rope")
    return out


def verify_drafts(starts, parents, tokens, target, draft, uniforms, path, kept, next, stream=None):
    """Which drafts stay: a walk down each request's tree that tests children against the target's probabilities with the given random numbers
    (include/turboquant_c/turboquant_b200.h, tq_verify_drafts).  starts int32 [n + 1] (what `plan` gives), parents and tokens int32 [rows], target and
    draft (or None: chosen drafts) fp32 or fp16 [rows, vocab], uniforms fp32 [rows].  Fills path [n, width], kept [n] and next [n], int32: what
    `PagedKVCache.keep` takes, and the tokens that follow."""
    _load_torch()
    on = _device_of(starts, "starts")
    try:
        n, width = path.shape
        rows, vocab = target.shape
        step, one = target.stride()
    except ValueError:
        raise ValueError("path must be [n, width], target [rows, vocab]") from None
    if (n | width | rows | vocab) > 0x7fffffff:
        raise ValueError("the sizes of path and target must fit in 32 bits")
    if _device_of(target, "target") != on:
        raise ValueError("target is on another device than starts")
    dp, drafted = None, 0
    if draft is not None:
        if draft.shape != target.shape or draft.dtype is not target.dtype:
            raise ValueError("target and draft must have the same shape and type")
        if _device_of(draft, "draft") != on:
            raise ValueError("draft is on another device than starts")
        drafted, other = draft.stride()
        if other != 1:
            one = other
        dp = draft.data_ptr()
    if one != 1 and vocab > 1:
        raise ValueError("rows of target and draft must be contiguous")
    if rows <= 1:      # (a stride that is not used may be anything)
        step, drafted = max(step, vocab), max(drafted, vocab)
    if uniforms.dtype is not _float32 or uniforms.numel() != rows or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be contiguous float32 [{rows}]")
    if _device_of(uniforms, "uniforms") != on:
        raise ValueError("uniforms are on another device than starts")
    if _lib.load().tq_verify_drafts(_ints(starts, "starts", n + 1, on), _ints(parents, "parents", rows, on), _ints(tokens, "tokens", rows, on), n, rows, target.data_ptr(),
                                    dp, TQ_F32 if target.dtype is _float32 else _tag(target, "verify_drafts"), vocab, step, drafted, uniforms.data_ptr(),
                                    _ints(path, "path", n * width, on), width, _ints(kept, "kept", n, on), _ints(next, "next", n, on),
                                    None if stream is None else _stream_ptr(stream)):
        check(-1, "verify_drafts")

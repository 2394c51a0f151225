"""Keys and values of many sequences in pages of one cache (``csrc/rotary.hip``,
``csrc/sattn.hip``).

A batch packs the new tokens of ``S`` sequences into the rows of ``[T, heads, D]``
tensors: those of sequence ``s`` are the rows ``starts[s] .. starts[s + 1]`` and the last
of its ``lengths[s]`` states; rows from ``starts[S]`` on belong to no sequence (a batch
padded to a captured graph's size).  State ``j`` of a sequence lies in page
``tables[s, j // page]`` at place ``j % page``.  ``tables`` [S, width], ``starts`` [S + 1]
(ascending from 0) and ``lengths`` [S] are int32 on the GPU and read by the kernels alone,
so nothing waits for the host and a captured call replays with new ones.  A table entry
that is no page of the cache holds no state: it is neither written nor read.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native
from .activations import _DTYPES as _WEIGHT_DTYPES, host_path
from .attention import _device_supported
from .rotary import _MAX_HEADS, _MAX_TOKENS, _weight_type, check_rotation, rotation_operands
from .window_attention import check_limits, host_limits, limits

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # TPF_BF16, TPF_F16
_MAX_HEAD_DIM = 128
_MAX_STATES = 1 << 30  # of a cache or of a table's row


class PagedCache:
    """``pages`` pages of ``page`` states: ``k`` and ``v`` are [pages, kv_heads, page,
    head_dim], BF16 or FP16 (head_dim a multiple of 8 up to 128)."""

    __slots__ = ("_k", "_v")

    def __init__(self, pages: int, kv_heads: int, page: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        shape = (pages, kv_heads, page, head_dim)
        self._take(*(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)))

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedCache":
        """A cache on the caller's tensors, which are used as they are."""
        cache = cls.__new__(cls)
        cache._take(k, v)
        return cache

    def _take(self, k, v) -> None:
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or t.ndim != 4:
                raise ValueError(f"a cache's {name} must be [pages, kv_heads, page, head_dim]")
            if t.dtype not in _DTYPES or t.shape != k.shape or t.dtype != k.dtype or t.device != k.device:
                raise ValueError("a cache's k and v must be alike, BF16 or FP16")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("a cache's tensors must be contiguous, on 16 bytes")
            if t.requires_grad:
                raise ValueError("no gradients pass through a cache")
        _, heads, page, D = k.shape
        if heads < 1 or page < 1 or D < 8 or D % 8 or D > _MAX_HEAD_DIM:
            raise ValueError("a cache needs kv heads, places on a page and a head dimension "
                             "that is a multiple of 8 up to 128")
        if k.numel() // D > _MAX_STATES:
            raise ValueError("a cache holds 2^30 states of all kv heads at most")
        self._k, self._v = k, v

    @property
    def k(self) -> torch.Tensor:
        return self._k

    @property
    def v(self) -> torch.Tensor:
        return self._v

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]


class _Batch(ctypes.Structure):  # tpf_paged_batch
    _fields_ = [(n, ctypes.c_void_p) for n in ("tables", "starts", "lengths")] + [
        (n, ctypes.c_int64) for n in ("S", "T", "width", "table_stride", "page", "pages")]


_AppendShape = ctypes.c_int64 * 14  # tpf_append_shape


def check_batch(unsupported, cache, tables, starts, lengths, tokens) -> None:
    """Arguments of a call on a cache; ``tokens``: (name, tensor, its heads or None)."""
    if not isinstance(cache, PagedCache):
        raise unsupported("needs a PagedCache")
    for name, t, dims in (("tables", tables, 2), ("starts", starts, 1), ("lengths", lengths, 1)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.ndim != dims:
            raise unsupported(f"{name} must be an int32 tensor of {dims} ax{'es' if dims > 1 else 'is'}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise unsupported(f"{name} must be contiguous along its last axis")
    S = lengths.shape[0]
    if tables.shape[0] != S or starts.shape[0] != S + 1:
        raise unsupported("tables, starts and lengths must have S, S + 1 and S entries")
    if tables.shape[1] * cache.page > _MAX_STATES:
        raise unsupported("a table's row holds 2^30 states at most")
    T = tokens[0][1].shape[0] if isinstance(tokens[0][1], torch.Tensor) and tokens[0][1].ndim == 3 else -1
    for name, t, heads in tokens:
        if not isinstance(t, torch.Tensor) or t.ndim != 3 or t.shape[0] != T or t.shape[2] != cache.head_dim:
            raise unsupported(f"{name} must have shape [T, heads, {cache.head_dim}]")
        if heads is not None and t.shape[1] != heads:
            raise unsupported(f"{name} must have the cache's {heads} kv heads")
        if t.dtype != cache.k.dtype:
            raise unsupported(f"{name} must have the cache's type")
        if t.requires_grad and torch.is_grad_enabled():
            raise unsupported("no gradients pass through a cache: call it under torch.no_grad()")
    if len({t.device for t in (cache.k, tables, starts, lengths, *(t for _, t, _ in tokens))}) != 1:
        raise unsupported("the cache, its tables and the tokens must share one device")
    if T > _MAX_TOKENS or any(t.shape[1] > _MAX_HEADS for _, t, _ in tokens):
        raise unsupported("at most 65535 heads and 2^26 - 32 tokens")


def batch_struct(k_cache, tables, starts, lengths, T: int) -> _Batch:
    S, width = tables.shape
    return _Batch(_native.ptr(tables), _native.ptr(starts), _native.ptr(lengths), S, T, width,
                  tables.stride(0) if S > 1 else width, k_cache.shape[2], k_cache.shape[0])


def _append_unsupported(reason: str):
    return ValueError(f"unsupported append case: {reason}")


class _AppendFn(torch.autograd.Function):
    """A Function, so that forward-mode AD and function transforms, which the native call
    would hide, are refused."""

    @staticmethod
    def forward(ctx, q, k, v, k_cache, v_cache, tables, starts, lengths, freq, qw, kw, eps, interleaved):
        T, Hk, D = k.shape
        H = 0 if q is None else q.shape[1]
        out = torch.empty((T, H, D), device=k.device, dtype=k.dtype)
        strides = [s if n > 1 else 0 for t in (k if q is None else q, k, v)
                   for n, s in zip(t.shape[:2], t.stride())]
        shape = _AppendShape(H, Hk, D, 0 if freq is None else len(freq), _DTYPES[k.dtype],
                             _WEIGHT_DTYPES[_weight_type(qw, kw)],
                             int(eps is not None), int(interleaved), *strides)
        ptr = _native.ptr
        with _native.device_ctx(k.device):
            _native.call("tpf_paged_append", ptr(q), ptr(k), ptr(v), ptr(freq), ptr(qw), ptr(kw),
                         0.0 if eps is None else eps, ptr(out), ptr(k_cache), ptr(v_cache), shape,
                         ctypes.byref(batch_struct(k_cache, tables, starts, lengths, T)),
                         _native.stream_of(k))
        ctx.mark_non_differentiable(out)
        return out

    @staticmethod
    def backward(ctx, d_out):  # pragma: no cover - nothing is differentiable
        raise RuntimeError("no gradients pass through a cache")


def append_kv(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, tables: torch.Tensor,
              starts: torch.Tensor, lengths: torch.Tensor, q: torch.Tensor | None = None,
              frequencies: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
              k_weight: torch.Tensor | None = None, eps: float | None = None,
              interleaved: bool = False) -> torch.Tensor | None:
    """Writes the new tokens' keys ``k`` and values ``v`` [T, kv_heads, D] to their places
    in ``cache`` (module text), in one launch with the norm and the rotation of
    ``qk_norm_rotary`` (by the states' numbers) on the keys' way and, where the new tokens'
    queries ``q`` [T, H, D] are given, on theirs: these are returned, contiguous, rows of
    no sequence as zeros.

    ``lengths`` count the new tokens.  Places of the cache that no new token has keep what
    they hold.  No two sequences may append to one page.  Other cases raise
    ``ValueError`` before any launch.
    """
    if (type(cache) is PagedCache
            and host_path(k, v, tables, starts, lengths, *(
                t for t in (q, frequencies, q_weight, k_weight) if t is not None))
            and (eps is None or type(eps) is float)):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().append_kv(cache._k, cache._v, k, v, tables, starts, lengths, q, frequencies,
                                       q_weight, k_weight, eps, bool(interleaved))
        if out is not None:
            return None if q is None else out
    tokens = [("k", k, None), ("v", v, None)] + ([] if q is None else [("q", q, None)])
    if isinstance(cache, PagedCache):
        tokens[0], tokens[1] = ("k", k, cache.kv_heads), ("v", v, cache.kv_heads)
    check_batch(_append_unsupported, cache, tables, starts, lengths, tokens)
    check_rotation(_append_unsupported, cache.head_dim, frequencies, q_weight, k_weight, eps, k.device)
    ok, reason = _device_supported(k)
    if not ok:
        raise _append_unsupported(reason)
    if torch.is_grad_enabled() and any(w is not None and w.requires_grad for w in (q_weight, k_weight)):
        raise _append_unsupported("no gradients pass through a cache: call it under torch.no_grad()")
    T = k.shape[0]
    if T == 0:
        return None if q is None else torch.empty_like(q, memory_format=torch.contiguous_format)
    freq, qw, kw = rotation_operands(frequencies, q_weight, k_weight)
    q, k, v = (t if t is None or t.stride(2) == 1 else t.contiguous() for t in (q, k, v))
    out = _AppendFn.apply(q, k, v, cache.k, cache.v, tables, starts, lengths, freq, qw, kw,
                          None if eps is None else float(eps), bool(interleaved))
    for t in (cache.k, cache.v):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)
    return None if q is None else out


def _attention_unsupported(reason: str):
    return ValueError(f"unsupported paged attention case: {reason}")


_PagedShape = ctypes.c_int64 * 8  # tpf_paged_shape


class _PagedFn(torch.autograd.Function):
    """A Function, so that forward-mode AD and function transforms, which the native call
    would hide, are refused."""

    @staticmethod
    def forward(ctx, q, k_cache, v_cache, tables, starts, lengths, window, sinks, scale):
        T, H, D = q.shape
        out = torch.empty((T, H, D), device=q.device, dtype=q.dtype)
        strides = (s if n > 1 else 0 for n, s in zip(q.shape[:2], q.stride()))
        shape = _PagedShape(H, k_cache.shape[1], D, _DTYPES[q.dtype], window, sinks, *strides)
        batch = ctypes.byref(batch_struct(k_cache, tables, starts, lengths, T))
        ws_bytes = int(_native.query("tpf_paged_attention_workspace_bytes", shape, batch))
        if ws_bytes < 0:
            raise _attention_unsupported(_native.query("tpf_last_error").decode(errors="replace"))
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes > 0 else None
        ptr = _native.ptr
        with _native.device_ctx(q.device):
            _native.call("tpf_paged_attention", ptr(q), ptr(k_cache), ptr(v_cache), ptr(out), ptr(ws),
                         ws_bytes, shape, batch, scale, _native.stream_of(q))
        ctx.mark_non_differentiable(out)
        return out

    @staticmethod
    def backward(ctx, d_out):  # pragma: no cover - nothing is differentiable
        raise RuntimeError("no gradients pass through a cache")


def paged_attention(q: torch.Tensor, cache: PagedCache, tables: torch.Tensor, starts: torch.Tensor,
                    lengths: torch.Tensor, window: int | None = None, sinks: int = 0,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of the new tokens' queries ``q`` [T, H, D] over their sequences' states in
    ``cache`` (module text; ``append_kv`` puts the new ones there): a token that is state
    ``p`` sees the states ``j <= p`` by the rules of ``window_attention``.  One new token
    for each sequence, chunks of them, or both at once.

    H is a multiple of the cache's kv heads; ``scale`` is 1/sqrt(D) unless given.  Returns
    [T, H, D], contiguous: a row that sees no state, or is of no sequence, is zeros.  Other
    cases raise ``ValueError`` before any launch.
    """
    if (type(cache) is PagedCache and host_path(q, tables, starts, lengths)
            and host_limits(window, sinks, scale)):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().paged_attention(q, cache._k, cache._v, tables, starts, lengths, window or 0,
                                             sinks, scale)
        if out is not None:
            return out
    check_batch(_attention_unsupported, cache, tables, starts, lengths, [("q", q, None)])
    check_limits(_attention_unsupported, window, sinks, scale)
    if q.shape[1] < 1 or q.shape[1] % cache.kv_heads:
        raise _attention_unsupported("the query heads must be a positive multiple of the kv heads")
    ok, reason = _device_supported(q)
    if not ok:
        raise _attention_unsupported(reason)
    if q.shape[0] == 0:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if (q.stride(2) != 1 or q.data_ptr() % 16
            or any(n > 1 and s % 8 for n, s in zip(q.shape[:2], q.stride()))):
        q = q.clone(memory_format=torch.contiguous_format)
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    return _PagedFn.apply(q, cache.k, cache.v, tables, starts, lengths, *limits(window, sinks), scale)


__all__ = ["PagedCache", "append_kv", "paged_attention"]

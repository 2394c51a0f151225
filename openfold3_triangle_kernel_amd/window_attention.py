"""Causal self-attention with a sliding window and sinks (``csrc/sattn.hip``,
``csrc/sattn_bwd.hip``).

    out_i = softmax_j(scale * q_i k_j) v_j  over the states j that token i sees

Token ``i`` sees the states ``j <= i`` with ``i - j < window`` or ``j < sinks`` that the key
mask leaves.  ``q`` is ``[*B, H, N, D]``; ``k`` and ``v`` are ``[*B, Hk, N, D]`` with ``H`` a
multiple of ``Hk`` (query head ``h`` reads kv head ``h // (H // Hk)``); the output is
``[*B, N, H, D]``, as cross attention's.  Operands are read in place as there.
"""

from __future__ import annotations

import ctypes
import math
import numbers

import torch

from . import _native
from .activations import differentiable_once, host_path
from .attention import _device_supported, shadow_enabled
from .cross_attention import _grad_like, _operand, _strides

_MAX_HEAD_DIM = 128
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # TPF_BF16, TPF_F16
_Shape = ctypes.c_int64 * 18  # tpf_window_shape


def _unsupported(reason: str):
    return ValueError(f"unsupported window attention case: {reason}")


def check_limits(unsupported, window, sinks, scale) -> None:
    """The arguments that ``window_attention`` and ``paged_attention`` share."""
    if window is not None and (not isinstance(window, numbers.Integral) or window < 1):
        raise unsupported("window must be a positive whole number or None")
    if not isinstance(sinks, numbers.Integral) or sinks < 0:
        raise unsupported("sinks must be a whole number from 0 on")
    if scale is not None and not (isinstance(scale, numbers.Real) and 1e-30 < scale < 1e30):
        raise unsupported("scale must be a number between 1e-30 and 1e30")


def host_limits(window, sinks, scale) -> bool:
    """Whether these arguments are of the kinds that the C++ host path takes."""
    return ((window is None or type(window) is int and 0 < window < 1 << 31) and type(sinks) is int
            and 0 <= sinks < 1 << 31 and (scale is None or type(scale) is float))


def limits(window, sinks) -> tuple[int, int]:
    """(window, sinks) as the native calls take them, 0 for no window."""
    most = 1 << 31  # (above every position)
    return (0, 0) if window is None else (min(int(window), most), min(int(sinks), most))


def _check(q, k, v, window, sinks, key_mask, scale) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise _unsupported(f"{name} must be a torch.Tensor")
        if t.ndim < 3:
            raise _unsupported(f"{name} must have shape [*B,H,N,D]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise _unsupported("q/k/v must share one type, BF16 or FP16")
    if k.shape != v.shape:
        raise _unsupported("k and v must have one shape")
    if q.shape[:-3] != k.shape[:-3] or q.shape[-2:] != k.shape[-2:]:
        raise _unsupported("q and k/v must share the batch prefix, the tokens and the head dimension")
    if not 1 <= q.shape[-1] <= _MAX_HEAD_DIM:
        raise _unsupported("requires 1<=D<=128")
    heads, kv_heads = q.shape[-3], k.shape[-3]
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise _unsupported("the query heads must be a positive multiple of the kv heads")
    check_limits(_unsupported, window, sinks, scale)
    tensors = [q, k, v]
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor) or key_mask.dtype != torch.bool:
            raise _unsupported("key_mask must be a boolean tensor")
        want = tuple(k.shape[:-3]) + (k.shape[-2],)
        try:
            fits = tuple(torch.broadcast_shapes(tuple(key_mask.shape), want)) == want
        except RuntimeError:
            fits = False
        if not fits or key_mask.ndim < 1 or key_mask.shape[-1] != k.shape[-2]:
            raise _unsupported("key_mask must broadcast to [*B,N]")
        tensors.append(key_mask)
    if len({t.device for t in tensors}) != 1:
        raise _unsupported("q/k/v and key_mask must share one device")
    if q.dtype != torch.bfloat16 and torch.is_grad_enabled() and any(
            t.requires_grad for t in (q, k, v)):
        raise _unsupported("gradients need BF16 operands")
    ok, reason = _device_supported(q)
    if not ok:
        raise _unsupported(reason)


def _mask_operand(mask: torch.Tensor | None, prefix, batch: int, N: int):
    """(bytes [batch or 1, N] or None, their batch stride) as the kernels read them."""
    if mask is None:
        return None, 0
    lead = mask.shape[:-1]
    if all(n == 1 for n in lead):
        return mask.reshape(N).contiguous(), 0
    if tuple(lead) != tuple(prefix):
        mask = mask.expand(tuple(prefix) + (N,))
    return mask.reshape(batch, N).contiguous(), N


def _shape(q, k, v, window, sinks, mask_stride):
    B, H, N, D = q.shape
    return _Shape(B, H, k.shape[1], N, D, _DTYPES[q.dtype], window, sinks, mask_stride, *_strides(q),
                  *_strides(k), *_strides(v))


def _forward(q, k, v, mask, mask_stride, window, sinks, scale, train, shadow=False):
    """(out, lse, what out's rounding drops); what is not asked for is None."""
    B, H, N, D = q.shape
    shape = _shape(q, k, v, window, sinks, mask_stride)
    ws_bytes = int(_native.query("tpf_window_forward_workspace_bytes", shape))
    if ws_bytes < 0 or (train and int(_native.query("tpf_window_backward_workspace_bytes", shape)) < 0):
        raise _unsupported(_native.query("tpf_last_error").decode(errors="replace"))
    out = torch.empty((B, N, H, D), device=q.device, dtype=q.dtype)
    lse = torch.empty((B, H, N), device=q.device, dtype=torch.float32) if train else None
    residual = torch.empty_like(out) if shadow else None
    ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes > 0 else None
    ptr = _native.ptr
    with _native.device_ctx(q.device):
        _native.call("tpf_window_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(mask),
                     out.data_ptr(), ptr(lse), ptr(residual), ptr(ws), ws_bytes, shape, scale,
                     _native.stream_of(q))
    return out, lse, residual


class _WindowFn(torch.autograd.Function):
    """Operands as the kernels read them: q [B, H, N, D], k and v [B, Hk, N, D]."""

    @staticmethod
    def forward(ctx, q, k, v, mask, mask_stride, window, sinks, scale, shadow):
        out, lse, residual = _forward(q, k, v, mask, mask_stride, window, sinks, scale, True, shadow)
        ctx.save_for_backward(q, k, v, mask, out, lse, residual)
        ctx.args = (mask_stride, window, sinks, scale)
        return out

    @staticmethod
    @differentiable_once
    def backward(ctx, d_out):
        q, k, v, mask, out, lse, residual = ctx.saved_tensors
        mask_stride, window, sinks, scale = ctx.args
        d_out = _native.aligned(d_out.to(q.dtype).contiguous())
        dq, dk, dv = (_grad_like(t) for t in (q, k, v))
        shape = _shape(q, k, v, window, sinks, mask_stride)
        grads = (ctypes.c_int64 * 9)(*_strides(dq), *_strides(dk), *_strides(dv))
        ws_bytes = int(_native.query("tpf_window_backward_workspace_bytes", shape))
        ws = torch.empty(max(ws_bytes, 16), device=q.device, dtype=torch.uint8)
        ptr = _native.ptr
        with _native.device_ctx(q.device):
            _native.call("tpf_window_backward_bf16", q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(mask),
                         out.data_ptr(), ptr(residual), d_out.data_ptr(), lse.data_ptr(), dq.data_ptr(),
                         dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, shape, grads, scale,
                         _native.stream_of(q))
        return dq, dk, dv, None, None, None, None, None, None


class _WindowInference(torch.autograd.Function):
    """The forward alone.  A Function all the same, so that forward-mode AD and function
    transforms, which the native calls would hide, are refused, and a trace records it."""

    @staticmethod
    def forward(ctx, q, k, v, mask, mask_stride, window, sinks, scale):
        return _forward(q, k, v, mask, mask_stride, window, sinks, scale, False)[0]

    @staticmethod
    def backward(ctx, d_out):  # pragma: no cover - only called without gradients
        raise RuntimeError("the inference call has no backward")


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int | None = None,
                     sinks: int = 0, key_mask: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Causal self-attention of ``q`` [*B, H, N, D] over ``k``, ``v`` [*B, Hk, N, D].

    Each token sees itself and the ``window - 1`` tokens before it (None: all of them) and
    the first ``sinks`` tokens up to itself.  ``key_mask``, boolean, broadcasts to [*B, N]:
    False drops the token as a state (it still has a row).  What a row does not see never
    reaches it, whatever K and V hold there; NaN and infinities that it sees do.  A row
    that sees nothing gives zeros, and zero gradients; one whose states all score -inf is
    NaN.  ``scale`` is 1/sqrt(D) unless given.  Returns ``[*B, N, H, D]`` of the operands'
    type.  BF16 operands have gradients (q, k, v); FP16 is for inference.  The policy of
    ``attention.shadow_enabled`` acts as in ``cross_attention``.  ``1 <= D <= 128`` (copied
    to a multiple of 8 where it is none).  Other cases raise ``ValueError`` before any
    launch.
    """
    if (host_path(q, k, v) and (key_mask is None or _native.host_eligible(key_mask))
            and host_limits(window, sinks, scale)):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().window_attention(q, k, v, window or 0, sinks, key_mask, scale)
        if out is not None:
            return out
    _check(q, k, v, window, sinks, key_mask, scale)
    head_dim = q.shape[-1]
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    prefix = q.shape[:-3]
    batch = math.prod(prefix)
    H, N = q.shape[-3], q.shape[-2]
    if batch == 0 or N == 0:
        out = torch.zeros(tuple(prefix) + (N, H, head_dim), device=q.device, dtype=q.dtype)
        edge = sum(t.reshape(-1)[:0].sum() for t in (q, k, v))
        return out + edge if edge.requires_grad else out
    pad = -head_dim % 8
    if pad:
        q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
    if q.ndim != 4:
        q, k, v = (t.reshape((batch,) + t.shape[-3:]) for t in (q, k, v))
    q, k, v = _operand(q), _operand(k), _operand(v)
    mask, mask_stride = _mask_operand(key_mask, prefix, batch, N)
    args = (mask, mask_stride, *limits(window, sinks), float(scale))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _WindowFn.apply(q, k, v, *args, shadow_enabled())
    else:
        out = _WindowInference.apply(q, k, v, *args)
    if pad:
        out = out[..., :head_dim].contiguous()
    return out if len(prefix) == 1 else out.reshape(tuple(prefix) + out.shape[1:])


__all__ = ["window_attention"]

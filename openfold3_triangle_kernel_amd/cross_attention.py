"""Cross attention to an encoder's states of another length (``csrc/xattn.hip``,
``csrc/xattn_bwd.hip``).

    out = softmax(scale * q k^T + key_mask) v

``q`` is ``[*B, H, Nq, D]``; ``k`` and ``v`` are ``[*B, Hk, Nk, D]`` with ``H`` a
multiple of ``Hk`` (query head ``h`` reads kv head ``h // (H // Hk)``); the output
is ``[*B, Nq, H, D]``, as the triangle attention's.  Head-major and
sequence-major operands, and other views whose channels are contiguous, are read
in place.  There is no pair bias: the mask is one entry per state, so all query
rows of a kv head see the same states and run as one row axis.
"""

from __future__ import annotations

import ctypes
import math
import numbers

import torch

from . import _native
from .activations import differentiable_once, host_path
from .attention import _device_supported, shadow_enabled

_MAX_HEAD_DIM = 128
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # TPF_BF16, TPF_F16
_MASK_NONE, _MASK_BYTES, _MASK_F32 = 0, 1, 2
_MAX_STATE_STRIDE = 1 << 23
_Shape = ctypes.c_int64 * 18  # tpf_xattn_shape


def _unsupported(reason: str):
    return ValueError(f"unsupported cross attention case: {reason}")


def _check(q, k, v, key_mask, scale) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise _unsupported(f"{name} must be a torch.Tensor")
        if t.ndim < 3:
            raise _unsupported(f"{name} must have shape [*B,H,N,D]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise _unsupported("q/k/v must share one type, BF16 or FP16")
    if k.shape != v.shape:
        raise _unsupported("k and v must have one shape")
    if q.shape[:-3] != k.shape[:-3] or q.shape[-1] != k.shape[-1]:
        raise _unsupported("q and k/v must share the batch prefix and the head dimension")
    if not 1 <= q.shape[-1] <= _MAX_HEAD_DIM:
        raise _unsupported("requires 1<=D<=128")
    heads, kv_heads = q.shape[-3], k.shape[-3]
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise _unsupported("the query heads must be a positive multiple of the kv heads")
    if scale is not None and not (isinstance(scale, numbers.Real) and 1e-30 < scale < 1e30):
        raise _unsupported("scale must be a number between 1e-30 and 1e30")
    tensors = [q, k, v]
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor):
            raise _unsupported("key_mask must be a torch.Tensor")
        if key_mask.dtype != torch.bool and not key_mask.is_floating_point():
            raise _unsupported("key_mask must be boolean or a floating additive mask")
        if key_mask.requires_grad:
            raise _unsupported("key_mask must not require gradients")
        want = tuple(k.shape[:-3]) + (k.shape[-2],)
        try:
            fits = tuple(torch.broadcast_shapes(tuple(key_mask.shape), want)) == want
        except RuntimeError:
            fits = False
        if not fits or key_mask.ndim < 1 or key_mask.shape[-1] != k.shape[-2]:
            raise _unsupported("key_mask must broadcast to [*B,Nk]")
        tensors.append(key_mask)
    if len({t.device for t in tensors}) != 1:
        raise _unsupported("q/k/v and key_mask must share one device")
    if q.dtype != torch.bfloat16 and torch.is_grad_enabled() and any(
            t.requires_grad for t in (q, k, v)):
        raise _unsupported("gradients need BF16 operands")
    ok, reason = _device_supported(q)
    if not ok:
        raise _unsupported(reason)


def _operand(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, H, N, D], or a contiguous copy where the kernels cannot read it."""
    # Strides of axes of one entry address nothing and may be anything.
    if (t.stride(3) == 1 and t.data_ptr() % 16 == 0
            and all(n <= 1 or s % 8 == 0 for n, s in zip(t.shape[:3], t.stride()))
            and (t.shape[2] <= 1 or t.stride(2) < _MAX_STATE_STRIDE)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _grad_like(t: torch.Tensor) -> torch.Tensor:
    """A gradient in the operand's storage order, where that keeps its channels
    contiguous (a broadcast operand's order may not)."""
    g = torch.empty_like(t)
    return g if g.stride(3) == 1 and all(s % 8 == 0 for s in g.stride()[:3]) else torch.empty(
        t.shape, device=t.device, dtype=t.dtype)


def _strides(t: torch.Tensor):
    sb, sh, sn, _ = t.stride()
    nb, nh, nn, _ = t.shape
    return (sb if nb > 1 else 0, sh if nh > 1 else 0, sn if nn > 1 else 0)


def additive_f32(mask: torch.Tensor) -> torch.Tensor:
    """An additive mask in FP32: finite values of FP64 stay finite."""
    if mask.dtype == torch.float64:
        ends = torch.finfo(torch.float32)
        mask = torch.where(torch.isfinite(mask), mask.clamp(ends.min, ends.max), mask)
    return mask.to(torch.float32)


def _mask_operand(mask: torch.Tensor | None, prefix, batch: int, Nk: int):
    """(tensor, kind, batch stride) of the mask as the kernels read it."""
    if mask is None:
        return None, _MASK_NONE, 0
    if mask.dtype == torch.bool:
        kind = _MASK_BYTES
    else:
        kind = _MASK_F32
        mask = additive_f32(mask)
    lead = mask.shape[:-1]
    if all(n == 1 for n in lead):
        return mask.reshape(Nk).contiguous(), kind, 0
    if tuple(lead) != tuple(prefix):
        mask = mask.expand(tuple(prefix) + (Nk,))
    return mask.reshape(batch, Nk).contiguous(), kind, Nk


def _shape(q, k, v, kind, mask_stride):
    B, H, Nq, D = q.shape
    _, Hk, Nk, _ = k.shape
    return _Shape(B, H, Hk, Nq, Nk, D, _DTYPES[q.dtype], kind, mask_stride, *_strides(q),
                  *_strides(k), *_strides(v))


def _workspace_bytes(shape, backward: bool) -> int:
    """Bytes of the forward's workspace; sizes that its launches (or the backward's) do
    not hold are refused."""
    ws_bytes = int(_native.query("tpf_xattn_forward_workspace_bytes", shape))
    if ws_bytes < 0 or (backward and int(
            _native.query("tpf_xattn_backward_workspace_bytes", shape)) < 0):
        raise _unsupported(_native.query("tpf_last_error").decode(errors="replace"))
    return ws_bytes


def _forward(q, k, v, mask, kind, mask_stride, scale, want_lse, shadow=False):
    """(out, lse, what out's rounding drops); what is not asked for is None."""
    B, H, Nq, D = q.shape
    shape = _shape(q, k, v, kind, mask_stride)
    ws_bytes = _workspace_bytes(shape, want_lse)
    out = torch.empty((B, Nq, H, D), device=q.device, dtype=q.dtype)
    lse = torch.empty((2 if kind == _MASK_F32 else 1, B, H, Nq), device=q.device,
                      dtype=torch.float32) if want_lse else None
    ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes > 0 else None
    residual = torch.empty_like(out) if shadow else None
    name, kept = ("tpf_xattn_forward", ()) if residual is None else (
        "tpf_xattn_forward_shadow_bf16", (residual.data_ptr(),))
    with _native.device_ctx(q.device):
        _native.call(name, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     _native.ptr(mask), out.data_ptr(), _native.ptr(lse), *kept, _native.ptr(ws),
                     ws_bytes, shape, scale, _native.stream_of(q))
    return out, lse, residual


class _CrossAttentionFn(torch.autograd.Function):
    """Operands as the kernels read them: q [B, H, Nq, D], k and v [B, Hk, Nk, D]."""

    @staticmethod
    def forward(ctx, q, k, v, mask, kind, mask_stride, scale, shadow):
        out, lse, residual = _forward(q, k, v, mask, kind, mask_stride, scale, True, shadow)
        ctx.save_for_backward(q, k, v, mask, out, lse, residual)
        ctx.args = (kind, mask_stride, scale)
        return out

    @staticmethod
    @differentiable_once
    def backward(ctx, d_out):
        q, k, v, mask, out, lse, residual = ctx.saved_tensors
        kind, mask_stride, scale = ctx.args
        d_out = _native.aligned(d_out.to(q.dtype).contiguous())
        dq, dk, dv = (_grad_like(t) for t in (q, k, v))
        shape = _shape(q, k, v, kind, mask_stride)
        grads = (ctypes.c_int64 * 9)(*_strides(dq), *_strides(dk), *_strides(dv))
        ws_bytes = int(_native.query("tpf_xattn_backward_workspace_bytes", shape))
        ws = torch.empty(max(ws_bytes, 16), device=q.device, dtype=torch.uint8)
        name, kept = ("tpf_xattn_backward_bf16", ()) if residual is None else (
            "tpf_xattn_backward_shadow_bf16", (residual.data_ptr(),))
        with _native.device_ctx(q.device):
            _native.call(name, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         _native.ptr(mask), out.data_ptr(), *kept, d_out.data_ptr(), lse.data_ptr(),
                         dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes,
                         shape, grads, scale, _native.stream_of(q))
        return dq, dk, dv, None, None, None, None, None


class _CrossAttentionInference(torch.autograd.Function):
    """The forward alone.  A Function all the same, so that forward-mode AD and function
    transforms, which the native calls would hide, are refused, and a trace records it."""

    @staticmethod
    def forward(ctx, q, k, v, mask, kind, mask_stride, scale):
        return _forward(q, k, v, mask, kind, mask_stride, scale, False)[0]

    @staticmethod
    def backward(ctx, d_out):  # pragma: no cover - only called without gradients
        raise RuntimeError("the inference call has no backward")


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    key_mask: torch.Tensor | None = None,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of ``q`` [*B, H, Nq, D] to the states ``k``, ``v`` [*B, Hk, Nk, D].

    ``key_mask`` broadcasts to ``[*B, Nk]``: boolean (True takes the state) or
    additive floating (added to the scores in 32 bits, finite values as if within
    +-1.5e38 ``scale``; -inf drops the state).  K and
    V of a dropped state are never used, whatever they hold; a NaN that is not dropped,
    in an additive mask too, reaches its rows.  A row without a state
    gives zeros, and zero gradients; one whose states all score -inf is NaN.  ``scale`` is 1/sqrt(D) unless given.  Returns
    ``[*B, Nq, H, D]`` of the operands' type.  BF16 operands have gradients (q, k, v);
    FP16 is for inference.  With the policy of ``attention.shadow_enabled`` (the default)
    a training forward also keeps what the output's rounding drops, a tensor of the
    output's size: no rounding of the output then enters the gradients, however much the
    states' values have in common.  ``1 <= D <= 128`` (copied to a multiple of 8 where it
    is none).  Other cases raise ``ValueError`` before any launch.
    """
    if (host_path(q, k, v) and (key_mask is None or _native.host_eligible(key_mask))
            and (scale is None or type(scale) in (float, int))):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().cross_attention(q, k, v, key_mask, scale)
        if out is not None:
            return out
    _check(q, k, v, key_mask, scale)
    head_dim = q.shape[-1]
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    prefix = q.shape[:-3]
    batch = math.prod(prefix)
    H, Nq = q.shape[-3], q.shape[-2]
    Nk = k.shape[-2]
    if batch == 0 or Nq == 0 or Nk == 0:
        # No row, or rows without a state: zeros, in the graph through empty slices.
        out = torch.zeros(tuple(prefix) + (Nq, H, head_dim), device=q.device, dtype=q.dtype)
        edge = sum(t.reshape(-1)[:0].sum() for t in (q, k, v))
        return out + edge if edge.requires_grad else out
    pad = -head_dim % 8
    if pad:
        q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
    if q.ndim != 4:
        q, k, v = (t.reshape((batch,) + t.shape[-3:]) for t in (q, k, v))
    q, k, v = _operand(q), _operand(k), _operand(v)
    mask, kind, mask_stride = _mask_operand(key_mask, prefix, batch, Nk)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _CrossAttentionFn.apply(q, k, v, mask, kind, mask_stride, float(scale),
                                      shadow_enabled())
    else:
        out = _CrossAttentionInference.apply(q, k, v, mask, kind, mask_stride, float(scale))
    if pad:
        out = out[..., :head_dim].contiguous()
    return out if len(prefix) == 1 else out.reshape(tuple(prefix) + out.shape[1:])


__all__ = ["cross_attention"]

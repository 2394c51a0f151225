"""Norms of queries and keys for each head with the rotation by position, in one pass
(``csrc/rotary.hip``).

    x^ = x / sqrt(mean(x^2) + eps),  z = x^ * w,  t_c = position * frequencies[c]
    y_a = z_a cos t_c - z_b sin t_c,  y_b = z_b cos t_c + z_a sin t_c

over the pairs (a, b) of a head's first ``2 * len(frequencies)`` channels: ``(c, c + half)``
or, interleaved, ``(2c, 2c + 1)``; the other channels are ``z``.  Scaling for long contexts
is in the frequencies, which are the caller's.
"""

from __future__ import annotations

import ctypes
import math
import numbers

import torch

from . import _native
from .activations import _DTYPES, differentiable_once, host_path
from .attention import _device_supported

_MAX_HEAD_DIM = 256
_MAX_HEADS, _MAX_TOKENS = 65535, (1 << 26) - 32  # (of a launch)
_Shape = ctypes.c_int64 * 25  # tpf_rotary_shape


def _unsupported(reason: str):
    return ValueError(f"unsupported rotary case: {reason}")


def check_rotation(unsupported, D: int, frequencies, q_weight, k_weight, eps, device) -> None:
    """The arguments that ``qk_norm_rotary`` and ``append_kv`` share."""
    if frequencies is not None:
        if (not isinstance(frequencies, torch.Tensor) or frequencies.ndim != 1
                or not frequencies.is_floating_point()):
            raise unsupported("frequencies must be a floating tensor of one axis")
        if 2 * frequencies.shape[0] > D:
            raise unsupported("more pairs of channels than the head has")
        if frequencies.requires_grad:
            raise unsupported("frequencies must not require gradients")
        if frequencies.device != device:
            raise unsupported("frequencies must lie on the operands' device")
    if eps is None:
        if q_weight is not None or k_weight is not None:
            raise unsupported("weights belong to a norm: give eps")
        return
    if not isinstance(eps, numbers.Real) or not 0.0 <= eps < 1e30:
        raise unsupported("eps must be a number between 0 and 1e30")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or tuple(w.shape) != (D,) or w.dtype not in _DTYPES:
            raise unsupported(f"{name} must be a BF16, FP16 or FP32 tensor of shape ({D},)")
        if w.device != device:
            raise unsupported(f"{name} must lie on the operands' device")


def rotation_operands(frequencies, q_weight, k_weight):
    """(frequencies in 64 bits or None, the weights, contiguous and of one type)."""
    if frequencies is not None:
        frequencies = frequencies.to(torch.float64).contiguous() if len(frequencies) else None
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        q_weight, k_weight = q_weight.float(), k_weight.float()
    return frequencies, q_weight, k_weight


def _check(q, k, positions, frequencies, q_weight, k_weight, eps) -> None:
    for name, t in (("q", q), ("k", k)):
        if not isinstance(t, torch.Tensor) or t.ndim < 3:
            raise _unsupported(f"{name} must be a torch.Tensor of shape [*B,H,N,D]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise _unsupported("q and k must share one type, BF16, FP16 or FP32")
    if q.shape[:-3] != k.shape[:-3] or q.shape[-2:] != k.shape[-2:]:
        raise _unsupported("q and k must share the batch prefix, the positions and the head dimension")
    D = q.shape[-1]
    if not 1 <= D <= _MAX_HEAD_DIM:
        raise _unsupported("requires 1<=D<=256")
    if max(q.shape[-3], k.shape[-3]) > _MAX_HEADS or math.prod(q.shape[:-3]) * q.shape[-2] > _MAX_TOKENS:
        raise _unsupported("at most 65535 heads and 2^26 - 32 tokens")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            raise _unsupported("positions must be int32 or int64")
        want = tuple(q.shape[:-3]) + (q.shape[-2],)
        try:
            fits = tuple(torch.broadcast_shapes(tuple(positions.shape), want)) == want
        except RuntimeError:
            fits = False
        if not fits:
            raise _unsupported("positions must broadcast to [*B,N]")
        if positions.device != q.device:
            raise _unsupported("positions must lie on the operands' device")
    if k.device != q.device:
        raise _unsupported("q and k must share one device")
    check_rotation(_unsupported, D, frequencies, q_weight, k_weight, eps, q.device)
    ok, reason = _device_supported(q)
    if not ok:
        raise _unsupported(reason)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, H, N, D] with contiguous channels (a copy where they are not)."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _like(t: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(t)
    return out if out.stride(3) == 1 else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _strides(t: torch.Tensor):
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()))


def _shape(q, k, out_q, out_k, positions, half, wtype, norm, interleaved):
    B, H, N, D = q.shape
    bits, step = 64, (0, 0)
    if positions is not None:
        bits = 64 if positions.dtype == torch.int64 else 32
        step = tuple(s if n > 1 else 0 for n, s in zip(positions.shape, positions.stride()))
    return _Shape(B, N, H, k.shape[1], D, half, _DTYPES[q.dtype], _DTYPES[wtype], int(norm),
                  int(interleaved), bits, *step, *_strides(q), *_strides(k), *_strides(out_q),
                  *_strides(out_k))


def _weight_type(qw, kw):
    return torch.float32 if qw is None and kw is None else (kw if qw is None else qw).dtype


def _forward(q, k, positions, freq, qw, kw, eps, interleaved):
    out_q, out_k = _like(q), _like(k)
    shape = _shape(q, k, out_q, out_k, positions, 0 if freq is None else len(freq),
                   _weight_type(qw, kw), eps is not None, interleaved)
    ptr = _native.ptr
    with _native.device_ctx(q.device):
        _native.call("tpf_rotary_forward", ptr(q), ptr(k), ptr(positions), ptr(freq), ptr(qw), ptr(kw),
                     0.0 if eps is None else eps, ptr(out_q), ptr(out_k), shape, _native.stream_of(q))
    return out_q, out_k


class _RotaryFn(torch.autograd.Function):
    """q [B, H, N, D] and k [B, Hk, N, D]; the last tensors are the operands as the kernel
    reads them, the weights before them as the graph knows them."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, freq, qw, kw, eps, interleaved):
        out = _forward(q, k, positions, freq, qw, kw, eps, interleaved)
        kept = (None, None) if eps is None else (q, k)
        ctx.save_for_backward(*kept, positions, freq, qw, kw)
        ctx.args = (eps, interleaved, tuple(None if w is None else w.dtype for w in (q_weight, k_weight)))
        return out

    @staticmethod
    @differentiable_once
    def backward(ctx, dy_q, dy_k):
        q, k, positions, freq, qw, kw = ctx.saved_tensors
        eps, interleaved, wtypes = ctx.args
        dy_q, dy_k = _rows(dy_q), _rows(dy_k)
        dq, dk = (_like(d if x is None else x) for d, x in ((dy_q, q), (dy_k, k)))
        wtype = _weight_type(qw, kw)
        want = ctx.needs_input_grad[2:4]
        dw = [torch.empty(dq.shape[3], device=dq.device, dtype=wtype) if w else None for w in want]
        shape = _shape(dy_q if q is None else q, dy_k if k is None else k, dq, dk, positions,
                       0 if freq is None else len(freq), wtype, eps is not None, interleaved)
        ws, ws_bytes = None, 0
        if any(want):
            ws_bytes = int(_native.query("tpf_rotary_backward_workspace_bytes", shape))
            ws = torch.empty(max(ws_bytes, 16), device=dq.device, dtype=torch.uint8)
        ptr = _native.ptr
        with _native.device_ctx(dq.device):
            _native.call("tpf_rotary_backward", ptr(q), ptr(k), ptr(dy_q), ptr(dy_k), ptr(positions),
                         ptr(freq), ptr(qw), ptr(kw), 0.0 if eps is None else eps, ptr(dq), ptr(dk),
                         ptr(dw[0]), ptr(dw[1]), ptr(ws), ws_bytes, shape,
                         (ctypes.c_int64 * 6)(*_strides(dy_q), *_strides(dy_k)), _native.stream_of(dq))
        dw = [None if w is None else w.to(t) for w, t in zip(dw, wtypes)]
        return dq, dk, *dw, None, None, None, None, None, None


class _RotaryInference(torch.autograd.Function):
    """The forward alone.  A Function all the same, so that forward-mode AD and function
    transforms, which the native calls would hide, are refused, and a trace records it."""

    @staticmethod
    def forward(ctx, q, k, positions, freq, qw, kw, eps, interleaved):
        return _forward(q, k, positions, freq, qw, kw, eps, interleaved)

    @staticmethod
    def backward(ctx, dy_q, dy_k):  # pragma: no cover - only called without gradients
        raise RuntimeError("the inference call has no backward")


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor | None = None,
                   frequencies: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float | None = None,
                   interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``q`` [*B, H, N, D] and ``k`` [*B, Hk, N, D] (BF16, FP16 or FP32, D up to 256), each
    head normalised and turned by its position: new tensors of their types and storage orders.

    ``eps`` None leaves the norm out; ``q_weight`` and ``k_weight`` [D] (BF16, FP16 or FP32)
    scale the normalised heads.  ``frequencies`` [half] are radians a position (kept in 64
    bits; None leaves the rotation out), ``positions`` whole numbers that broadcast to
    [*B, N] (None: 0 .. N - 1); while position times frequency is below 2^28 radians, an
    angle is within 2^-22 of it.  Statistics and products are in 32 bits.  Gradients: q, k and the weights.  Other cases raise
    ``ValueError`` before any launch.
    """
    if (host_path(q, k, *(t for t in (positions, frequencies, q_weight, k_weight) if t is not None))
            and (eps is None or type(eps) is float)):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().qk_norm_rotary(q, k, positions, frequencies, q_weight, k_weight, eps,
                                            bool(interleaved))
        if out is not None:
            return out
    _check(q, k, positions, frequencies, q_weight, k_weight, eps)
    if q.numel() + k.numel() == 0:
        edge = sum(w.reshape(-1)[:0].sum() for w in (q_weight, k_weight) if w is not None)
        return tuple(t.clone() if isinstance(edge, int) else t + edge.to(t.dtype) for t in (q, k))
    prefix, N = q.shape[:-3], q.shape[-2]
    batch = math.prod(prefix)
    if positions is not None:
        positions = positions.expand(tuple(prefix) + (N,)).reshape(batch, N)
    freq, qw, kw = rotation_operands(frequencies, q_weight, k_weight)
    q4, k4 = (t if t.ndim == 4 else t.reshape((batch,) + t.shape[-3:]) for t in (q, k))
    q4, k4 = _rows(q4), _rows(k4)
    eps = None if eps is None else float(eps)
    grad = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, q_weight, k_weight))
    if grad:
        qw, kw = (None if w is None else w.detach() for w in (qw, kw))
        out = _RotaryFn.apply(q4, k4, q_weight, k_weight, positions, freq, qw, kw, eps, bool(interleaved))
    else:
        out = _RotaryInference.apply(q4, k4, positions, freq, qw, kw, eps, bool(interleaved))
    if len(prefix) == 1:
        return out
    return tuple(o.reshape(t.shape) for o, t in zip(out, (q, k)))


__all__ = ["qk_norm_rotary"]

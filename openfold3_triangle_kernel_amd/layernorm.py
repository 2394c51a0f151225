"""LayerNorm with FP32 statistics.

``layer_norm`` (``csrc/norm.hip``): BF16, FP16 or FP32 rows of any channel count,
parameters of any of these types, its backward from the rows or from their
normalised values in 8 bits.

``layer_norm_bf16`` (``csrc/layernorm.hip``): BF16 pair rows read through the strides
of a pair grid.

Replaces the torch LayerNorm that OpenFold3's pair-stack modules apply to
their input (``openfold3/core/model/primitives/normalization.py:54-78``:
statistics and affine in FP32, result in the input dtype).  The kernel reads
the rows of a ``[*, I, J, C]`` tensor through its strides, so the transposed
view of the ending-node module is normalised without a copy; the output is
contiguous.  The backward writes dx with the input's own strides and forms
dgamma / dbeta from fixed-order partial sums (deterministic).
"""

from __future__ import annotations

import torch

from . import _native
from .activations import _DTYPES, as_rows, check_rows, code_buffers, differentiable_once, host_path
from .attention import _device_ctx


def _grid_view(x: torch.Tensor) -> torch.Tensor:
    """x as a 4-D [B, I, J, C] view (a copy only when the strides do not allow
    one), channels contiguous, row strides multiples of 8 elements."""
    C = x.shape[-1]
    if x.dim() == 1:
        x = x.reshape(1, 1, 1, C)
    elif x.dim() < 4:
        x = x.reshape((1,) * (4 - x.dim()) + tuple(x.shape))
    elif x.dim() > 4:
        try:
            x = x.view(-1, *x.shape[-3:])
        except RuntimeError:
            x = x.reshape(-1, *x.shape[-3:])
    if (x.stride(-1) != 1 or any(s % 8 for s in x.stride()[:3]) or x.data_ptr() % 16
            or any(s < 0 for s in x.stride())):
        x = x.contiguous()
    return x


def _strides(t: torch.Tensor):
    # A size-1 dimension's stride is never used to address anything.
    return [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]


class _LayerNormBf16(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        shape = x.shape
        x4 = _grid_view(x)
        B, I, J, C = x4.shape
        dev = x.device
        w = None if weight is None else weight.detach().float().contiguous()
        b = None if bias is None else bias.detach().float().contiguous()
        y = torch.empty((B, I, J, C), device=dev, dtype=torch.bfloat16)
        mean = torch.empty(B * I * J, device=dev, dtype=torch.float32)
        rstd = torch.empty_like(mean)
        with _device_ctx(dev):
            _native.call("tpf_layer_norm_forward_bf16", x4.data_ptr(), B, I, J, *_strides(x4), C,
                         None if w is None else w.data_ptr(), None if b is None else b.data_ptr(),
                         float(eps), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                         _native.stream_of(x4))
        ctx.save_for_backward(x4, mean, rstd, w)
        ctx.shape = shape
        ctx.param_dtypes = (None if weight is None else weight.dtype,
                            None if bias is None else bias.dtype)
        ctx.set_materialize_grads(False)
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        x4, mean, rstd, w = ctx.saved_tensors
        B, I, J, C = x4.shape
        dev = x4.device
        dy = dy.reshape(B * I * J, C).to(torch.bfloat16).contiguous()
        dx = torch.empty_like(x4)
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dw = db = ws = None
        ws_bytes = 0
        if want:
            dw = torch.empty(C, device=dev, dtype=torch.float32)
            db = torch.empty(C, device=dev, dtype=torch.float32)
            ws_bytes = int(_native.query("tpf_layer_norm_backward_workspace_bytes", B * I * J, C))
            ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        with _device_ctx(dev):
            _native.call("tpf_layer_norm_backward_bf16", dy.data_ptr(), x4.data_ptr(), B, I, J,
                         *_strides(x4), *_strides(dx), C, mean.data_ptr(), rstd.data_ptr(),
                         None if w is None else w.data_ptr(), dx.data_ptr(),
                         None if dw is None else dw.data_ptr(),
                         None if db is None else db.data_ptr(),
                         None if ws is None else ws.data_ptr(), ws_bytes, _native.stream_of(dy))
        gw = gb = None
        if ctx.needs_input_grad[1] and ctx.param_dtypes[0] is not None:
            gw = dw.to(ctx.param_dtypes[0])
        if ctx.needs_input_grad[2] and ctx.param_dtypes[1] is not None:
            gb = db.to(ctx.param_dtypes[1])
        return dx.view(ctx.shape), gw, gb, None


def layer_norm_bf16(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
                    eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm over the last dimension of a CUDA BF16 tensor with FP32
    statistics and FP32 affine parameters; returns contiguous BF16."""
    if not (x.is_cuda and x.dtype == torch.bfloat16):
        raise ValueError("layer_norm_bf16 needs a CUDA bfloat16 tensor")
    C = x.shape[-1]
    if C % 8 or not 8 <= C <= 2048:
        raise ValueError("layer_norm_bf16 needs the channel count to be a multiple of 8 in [8, 2048]")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and tuple(p.shape) != (C,):
            raise ValueError(f"{name} must have shape ({C},)")
    if x.numel() == 0:
        raise ValueError("layer_norm_bf16 needs a nonempty tensor")
    return _LayerNormBf16.apply(x, weight, bias, eps)


def _norm_forward(x2, w, b, eps, save):
    """(y, mean, rstd, codes, scales) of rows x2; what ``save`` does not ask for is None."""
    R, C = x2.shape
    dev = x2.device
    y = torch.empty((R, C), device=dev, dtype=x2.dtype)
    mean = torch.empty(R, device=dev, dtype=torch.float32) if save == "full" else None
    rstd = torch.empty(R, device=dev, dtype=torch.float32) if save else None
    codes, scales = code_buffers(R, C, dev) if save == "int8" else (None, None)
    p = w if w is not None else b
    ptr = _native.ptr
    with _device_ctx(dev):
        _native.call("tpf_norm_forward", x2.data_ptr(), x2.stride(0) if R > 1 else C, R, C,
                     _DTYPES[x2.dtype], ptr(w), ptr(b), 0 if p is None else _DTYPES[p.dtype], eps,
                     y.data_ptr(), ptr(mean), ptr(rstd), ptr(codes), ptr(scales),
                     _native.stream_of(x2))
    return y, mean, rstd, codes, scales


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, bias, w, b, eps, save):
        y, mean, rstd, codes, scales = _norm_forward(x2, w, b, eps, save)
        ctx.save_for_backward(x2 if save == "full" else None, mean, rstd, codes, scales, w)
        ctx.args = (x2.dtype, x2.shape, None if weight is None else weight.dtype,
                    None if bias is None else bias.dtype)
        return y

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        x2, mean, rstd, codes, scales, w = ctx.saved_tensors
        dtype, (R, C), wtype, btype = ctx.args
        dev = dy.device
        dy = dy.to(dtype).contiguous()
        dx = torch.empty((R, C), device=dev, dtype=dtype)
        # The fold writes the gradients in the type of the weight as the forward read it
        # (FP32 beside a bias of another type): dx needs that weight, not a rounding of it.
        ptype = w.dtype if w is not None else torch.float32 if btype is None else btype
        dw = torch.empty(C, device=dev, dtype=ptype) if ctx.needs_input_grad[1] else None
        db = torch.empty(C, device=dev, dtype=ptype) if ctx.needs_input_grad[2] else None
        ws, ws_bytes = None, 0
        if dw is not None or db is not None:
            ws_bytes = int(_native.query("tpf_norm_backward_workspace_bytes", R, C))
            ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        ptr = _native.ptr
        with _device_ctx(dev):
            _native.call("tpf_norm_backward", dy.data_ptr(), ptr(x2),
                         0 if x2 is None else x2.stride(0) if R > 1 else C, ptr(codes), ptr(scales),
                         ptr(mean), rstd.data_ptr(), R, C, _DTYPES[dtype], ptr(w), _DTYPES[ptype],
                         dx.data_ptr(), C, ptr(dw), ptr(db), ptr(ws), ws_bytes,
                         _native.stream_of(dy))
        return (dx, None if dw is None else dw.to(wtype), None if db is None else db.to(btype), None,
                None, None, None)


class _LayerNormInference(torch.autograd.Function):
    """The forward alone.  A Function all the same, so that forward-mode AD and function
    transforms, which the native calls would hide, are refused, and a trace records it."""

    @staticmethod
    def forward(ctx, x2, w, b, eps):
        return _norm_forward(x2, w, b, eps, None)[0]

    @staticmethod
    def backward(ctx, dy):  # pragma: no cover - only called without gradients
        raise RuntimeError("the inference call has no backward")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5,
               save: str = "full") -> torch.Tensor:
    """LayerNorm over the last dimension of ``x`` [*, C] (BF16, FP16 or FP32, any C),
    with statistics and affine parameters in 32 bits; contiguous, of ``x``'s type.

    ``weight`` and ``bias`` [C] are BF16, FP16 or FP32 and may be None.  The backward
    reads ``x`` (``save="full"``) or, with ``save="int8"``, the normalised rows kept in 8
    bits a value (``compress_activation``'s form): its results are then the
    gradient's formula at the decoded values, and ``x`` is not kept.
    """
    if save not in ("full", "int8"):
        raise ValueError('save must be "full" or "int8"')
    if host_path(x, *(t for t in (weight, bias) if t is not None)):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().layer_norm(x, weight, bias, eps, save == "int8")
        if out is not None:
            return out
    check_rows("layer_norm", x)
    C = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if not isinstance(p, torch.Tensor) or tuple(p.shape) != (C,):
            raise ValueError(f"{name} must have shape ({C},)")
        if p.dtype not in _DTYPES or p.device != x.device:
            raise ValueError(f"{name} must be BF16, FP16 or FP32 on the input's device")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if x.numel() == 0:
        out = x
        for p, op in ((weight, torch.mul), (bias, torch.add)):
            out = out if p is None else op(out, p.to(x.dtype))
        return out.clone() if out is x else out
    w, b = (None if p is None else p.contiguous() for p in (weight, bias))
    if w is not None and b is not None and w.dtype != b.dtype:
        w, b = w.float(), b.float()
    grad = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, weight, bias))
    if grad:
        w, b = (None if p is None else p.detach() for p in (w, b))
        y = _LayerNormFn.apply(as_rows(x), weight, bias, w, b, float(eps), save)
    else:
        y = _LayerNormInference.apply(as_rows(x), w, b, float(eps))
    return y.view(x.shape)


__all__ = ["layer_norm", "layer_norm_bf16"]

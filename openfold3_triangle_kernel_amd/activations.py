"""Activations kept in 8 bits, and their use in the backward pass (``csrc/act8.hip``).

32 channels of a row share a power of two ``2^k``, ``k`` the smallest whole number
from -120 on for which ``round(max / 2^k)`` is at most 127 (and at most 121, 9 for
FP16: a larger quotient is held as 127, so decoded values are finite); a value ``x`` is held as
``round(x / 2^k)`` (ties to even) in one byte: 33/32 byte a value, an error of at
most 1/127.5 of the block's largest magnitude (or 2^-121, half the smallest step).  A decoded value has seven bits and is
exact in BF16, so the matrix cores take it as it is.  A block that holds an
infinity or NaN decodes to NaN.

``linear`` keeps its input that way for the gradient of its weight;
``layer_norm(..., save="int8")`` its normalised rows.
"""

from __future__ import annotations

import functools

import torch

from . import _native
from .attention import _device_supported, _is_gfx950

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # TPF_BF16, TPF_F16, TPF_F32
_BLOCK = 32
_GEMM_SPAN = (1 << 31) - 1  # bytes of a GEMM operand
_MAX_FEATURES = 1 << 23  # and elements between rows: 64 of them lie within 32-bit offsets


class CompressedActivation:
    """A tensor in 8 bits: ``codes`` uint8 [R, pitch] (128 + the rounded quotient;
    pitch: the channels rounded up to whole blocks), ``scales`` uint8
    [R, pitch / 32] (k + 127, 255 for a block that is not finite), and the
    ``shape`` and ``dtype`` of what it stands for."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, torch.Size(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def differentiable_once(backward):
    """The ``backward`` of a Function whose kernels have no second derivative: with
    ``create_graph`` its gradients raise when they are differentiated, instead of
    passing for constants."""

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        err = torch._C._functions.DelayedError(
            b"trying to differentiate twice a function that was marked with @once_differentiable",
            len(out))
        return err(*(t if t is None else t.detach().requires_grad_(True) for t in out))

    return wrapper


def host_path(*tensors) -> bool:
    """Whether a call on these tensors may be tried on the C++ host path."""
    return (_native.host_eligible(*tensors) and tensors[0].is_cuda
            and _is_gfx950(tensors[0].device) and _native.host() is not None)


def check_rows(what: str, x) -> None:
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{what} needs a torch.Tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} needs a BF16, FP16 or FP32 tensor")
    if x.ndim < 1 or x.shape[-1] < 1 or x.shape[-1] > 1 << 24:
        raise ValueError(f"{what} needs a tensor of 1 to 2^24 channels")
    ok, reason = _device_supported(x)
    if not ok:
        raise ValueError(f"{what}: {reason}")


def as_rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as [R, C] rows whose channels are contiguous (a copy only where its
    strides allow no view)."""
    x2 = x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(1) == 1 or x2.shape[1] == 1 else x2.contiguous()


def code_buffers(rows: int, channels: int, device):
    blocks = -(-channels // _BLOCK)
    return (torch.empty((rows, blocks * _BLOCK), device=device, dtype=torch.uint8),
            torch.empty((rows, blocks), device=device, dtype=torch.uint8))


def _pack(x2: torch.Tensor):
    R, C = x2.shape
    codes, scales = code_buffers(R, C, x2.device)
    if R:
        with _native.device_ctx(x2.device):
            _native.call("tpf_act8_pack", x2.data_ptr(), x2.stride(0), R, C, _DTYPES[x2.dtype],
                         codes.data_ptr(), scales.data_ptr(), _native.stream_of(x2))
    return codes, scales


class _PackFn(torch.autograd.Function):
    """The codes and scales of rows x [R, C].  A Function for traces to record and function
    transforms to be refused; its outputs are whole numbers, without derivatives."""

    @staticmethod
    def forward(ctx, x2):
        codes, scales = _pack(x2)
        ctx.mark_non_differentiable(codes, scales)
        return codes, scales


class _UnpackFn(torch.autograd.Function):
    """The tensor of ``shape`` and ``dtype`` that codes and scales stand for."""

    @staticmethod
    def forward(ctx, codes, scales, shape, dtype):
        out = torch.empty(shape, device=codes.device, dtype=dtype)
        if out.numel():
            C = shape[-1]
            with _native.device_ctx(out.device):
                _native.call("tpf_act8_unpack", codes.data_ptr(), scales.data_ptr(),
                             out.numel() // C, C, out.data_ptr(), C, _DTYPES[dtype],
                             _native.stream_of(out))
        return out


def compress_activation(x: torch.Tensor) -> CompressedActivation:
    """``x`` [*, C] (BF16, FP16 or FP32) in 8 bits; no gradient passes through."""
    if host_path(x):
        # The common form entirely in C++; None (nothing launched) for any other.
        packed = _native.host().act8_pack(x)
        if packed is not None:
            return CompressedActivation(*packed, x.shape, x.dtype)
    check_rows("compress_activation", x)
    return CompressedActivation(*_PackFn.apply(as_rows(x.detach())), x.shape, x.dtype)


def decompress_activation(saved: CompressedActivation,
                          dtype: torch.dtype | None = None) -> torch.Tensor:
    """The tensor that ``saved`` stands for, in its own type or ``dtype``."""
    if not isinstance(saved, CompressedActivation):
        raise ValueError("decompress_activation needs a CompressedActivation")
    dtype = saved.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError("decompress_activation gives BF16, FP16 or FP32")
    if host_path(saved.codes, saved.scales):
        out = _native.host().act8_unpack(saved.codes, saved.scales, saved.shape, dtype)
        if out is not None:
            return out
    if not saved.shape or saved.shape[-1] < 1:
        raise ValueError("decompress_activation: the shape has no channels")
    C = saved.shape[-1]
    rows = saved.shape.numel() // C
    blocks = -(-C // _BLOCK)
    for t, width in ((saved.codes, blocks * _BLOCK), (saved.scales, blocks)):
        if t.dtype != torch.uint8 or tuple(t.shape) != (rows, width) or not t.is_contiguous():
            raise ValueError("decompress_activation: codes or scales do not fit the shape")
    if saved.codes.device != saved.scales.device:
        raise ValueError("decompress_activation: codes and scales on different devices")
    ok, reason = _device_supported(saved.codes)
    if not ok:
        raise ValueError(f"decompress_activation: {reason}")
    shape = tuple(map(int, saved.shape))  # (tensors in a trace)
    return _UnpackFn.apply(saved.codes, saved.scales, shape, dtype)


def _row_gemm(a: torch.Tensor, b: torch.Tensor, b_kc: bool) -> torch.Tensor:
    """``a [R, K] @ b.t()`` (b_kc: b [N, K]) or ``a @ b`` (b [K, N]) on the BF16 GEMM;
    rows beyond an operand's 2 GiB in further calls (a row's result does not depend
    on the row count)."""
    R, K = map(int, a.shape)  # (tensors in a trace)
    N = int(b.shape[0] if b_kc else b.shape[1])
    out = torch.empty((R, N), device=a.device, dtype=torch.bfloat16)
    ld = int(a.stride(0)) if R > 1 else K
    step = max(1, _GEMM_SPAN // (2 * ld))
    with _native.device_ctx(a.device):
        for r in range(0, R, step):
            n = min(step, R - r)
            _native.call("tpf_row_gemm_bf16", a.data_ptr() + 2 * r * ld, ld, b.data_ptr(), int(b_kc),
                         out.data_ptr() + 2 * r * N, n, N, K, _native.stream_of(a))
    return out


def _gemm_rows(x: torch.Tensor) -> torch.Tensor:
    """[R, C] rows as the GEMM reads them: 16-byte aligned rows of whole vectors, 64 of
    them within 32-bit offsets."""
    ld = x.stride(0)
    if x.stride(1) != 1 or (x.shape[0] > 1 and (ld % 8 or not x.shape[1] <= ld <= _MAX_FEATURES)):
        x = x.contiguous()
    return _native.aligned(x)


def weight_grad(dy: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, channels: int,
                dtype: torch.dtype) -> torch.Tensor:
    """dW [N, C] = dy^T x of BF16 rows dy [R, N] and x [R, C] in 8 bits."""
    R, N = dy.shape
    ld = dy.stride(0) if R > 1 else N
    out = torch.float32 if dtype == torch.float32 else torch.bfloat16
    dw = torch.empty((N, channels), device=dy.device, dtype=out)
    ws_bytes = int(_native.query("tpf_wgrad_act8_workspace_bytes", R, N, channels, ld))
    ws = torch.empty(ws_bytes, device=dy.device, dtype=torch.uint8) if ws_bytes > 0 else None
    with _native.device_ctx(dy.device):
        _native.call("tpf_wgrad_act8", dy.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), R, N,
                     channels, dw.data_ptr(), _DTYPES[out], _native.ptr(ws), max(ws_bytes, 0),
                     _native.stream_of(dy))
    return dw.to(dtype)


def _weight_grad_full(dy: torch.Tensor, x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """dW [N, K] = dy^T x of BF16 rows; rows beyond an operand's 2 GiB in further products,
    whose FP32 sums are added in order."""
    from .modules import _wgrad

    R, pitch = dy.shape[0], max(dy.stride(0), x.stride(0))
    step = max(1, _GEMM_SPAN // (2 * pitch))
    dw = _wgrad(dy[:step], x[:step], dtype if R <= step else torch.float32)
    for r in range(step, R, step):
        dw += _wgrad(dy[r:r + step], x[r:r + step], torch.float32)
    return dw.to(dtype)


class _LinearFn(torch.autograd.Function):
    """y = x w^T over rows x [R, K]; w [N, K] in its own type, used in BF16."""

    @staticmethod
    def forward(ctx, x, weight, save):
        w = _native.aligned(weight.detach().to(torch.bfloat16).contiguous())
        x = _gemm_rows(x.detach())
        ctx.save = save
        ctx.weight_dtype = weight.dtype
        kept = ()
        if ctx.needs_input_grad[1]:
            kept = _pack(x) if save == "int8" else (x,)
        ctx.save_for_backward(w, *kept)
        return _row_gemm(x, w, True)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        w, *kept = ctx.saved_tensors
        dy = _gemm_rows(dy.to(torch.bfloat16))
        dx = _row_gemm(dy, w, False) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            if ctx.save == "int8":
                dw = weight_grad(dy, *kept, w.shape[1], ctx.weight_dtype)
            else:
                dw = _weight_grad_full(dy, kept[0], ctx.weight_dtype)
        return dx, dw, None


def linear(x: torch.Tensor, weight: torch.Tensor, save: str = "int8") -> torch.Tensor:
    """``x`` [*, K] times ``weight``^T (``weight`` [N, K]) on the BF16 GEMM.

    For the gradient of ``weight`` the input is kept in 8 bits (``save="int8"``, about
    half of BF16; a channel below 1/255 of the largest among its 32 is kept as 0 and gives
    its column no gradient) or as it is (``"full"``).  ``x`` is BF16, ``weight`` BF16 or FP32 (used
    in BF16, its gradient from FP32 sums in its own type); K and N are multiples of 8 up
    to 2^23.
    """
    if save not in ("int8", "full"):
        raise ValueError('save must be "int8" or "full"')
    if save == "int8" and host_path(x, weight):
        # The common form entirely in C++; None (nothing launched) for any other.
        out = _native.host().linear(x, weight)
        if out is not None:
            return out
    check_rows("linear", x)
    if x.dtype != torch.bfloat16:
        raise ValueError("linear needs a BF16 input")
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError("linear needs a weight [N, K] for an input [*, K]")
    if weight.dtype not in (torch.bfloat16, torch.float32) or weight.device != x.device:
        raise ValueError("linear needs a BF16 or FP32 weight on the input's device")
    N, K = weight.shape
    if N < 8 or N % 8 or K % 8 or max(N, K) > _MAX_FEATURES or N * K * 2 > _GEMM_SPAN:
        raise ValueError("linear needs feature counts that are multiples of 8 up to 2^23, "
                         "the weight below 2 GiB")
    if x.numel() == 0:
        return x.matmul(weight.to(x.dtype).t())
    return _LinearFn.apply(x.reshape(-1, K), weight, save).view(x.shape[:-1] + (N,))


__all__ = ["CompressedActivation", "compress_activation", "decompress_activation", "linear"]

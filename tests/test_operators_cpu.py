"""Refusals of the cross-attention, layer-norm and 8-bit activation operators without a
GPU: host tensors and bad arguments raise before any native call, the C ABI answers
bad shapes with a status before any launch, and the block runs its formulas in
PyTorch on the CPU."""

import ctypes
import math

import pytest
import torch

from openfold3_triangle_kernel_amd import (
    CompressedActivation,
    CrossAttention,
    compress_activation,
    cross_attention,
    decompress_activation,
    layer_norm,
    linear,
    set_turbopairformer_strict,
    stock_invocation_count,
)


def _qkv(B=1, H=2, Hk=2, Nq=4, Nk=8, D=64, dtype=torch.bfloat16):
    return [torch.zeros(B, h, n, D, dtype=dtype) for h, n in ((H, Nq), (Hk, Nk), (Hk, Nk))]


@pytest.mark.parametrize("args,match", [
    ((*_qkv(),), "GPU"),
    ((_qkv()[0], _qkv()[1], None), "torch.Tensor"),
    ((*(t[0, 0] for t in _qkv()),), "shape"),
    ((*_qkv(dtype=torch.float32),), "BF16 or FP16"),
    ((*_qkv(D=129),), "D<=128"),
    ((*_qkv(H=3),), "multiple"),
    ((_qkv()[0], _qkv()[1], _qkv(Nk=9)[2]), "one shape"),
    ((_qkv(B=2)[0], *_qkv()[1:]), "batch prefix"),
    ((_qkv(D=32)[0], *_qkv()[1:]), "head dimension"),
    ((*_qkv(), torch.zeros(7)), "broadcast"),
    ((*_qkv(), torch.zeros(3, 8)), "broadcast"),
    ((*_qkv(), torch.zeros(1)), "broadcast"),
    ((*_qkv(), torch.zeros(8, dtype=torch.int64)), "boolean"),
    ((*_qkv(), torch.zeros(8, requires_grad=True)), "must not require"),
    ((*_qkv(), None, -1.0), "scale"),
    ((*_qkv(), None, float("nan")), "scale"),
])
def test_cross_attention_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        cross_attention(*args)


def test_rows_operators_refuse():
    x, w = torch.zeros(4, 16), torch.ones(16)
    for call, match in ((lambda: layer_norm(x, w), "GPU"),
                        (lambda: layer_norm(x.long()), "BF16"),
                        (lambda: layer_norm(x, save="fp8"), "save"),
                        (lambda: layer_norm(None), "torch.Tensor"),
                        (lambda: compress_activation(x), "GPU"),
                        (lambda: compress_activation(torch.tensor(1.0)), "channels"),
                        (lambda: decompress_activation(None), "CompressedActivation"),
                        (lambda: linear(x.bfloat16(), x.bfloat16()), "GPU"),
                        (lambda: linear(x, x, save="half"), "save")):
        with pytest.raises(ValueError, match=match):
            call()


def test_decompress_checks_what_it_is_given():
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    for args in ((codes, scales, (4, 33), torch.float32), (codes, scales[:3], (4, 20), torch.float32),
                 (codes.int(), scales, (4, 20), torch.float32), (codes, scales, (4, 0), torch.float32),
                 (codes, scales, (), torch.float32), (codes, scales, (4, 20), torch.int32),
                 (codes, scales, (4, 20), torch.float32)):
        with pytest.raises(ValueError):
            decompress_activation(CompressedActivation(*args))


def _shape(**kw):
    v = dict(B=1, H=2, Hk=2, Nq=4, Nk=8, D=64, dtype=0, kind=0, ms=0, q=(512, 256, 64),
             k=(1024, 512, 64), v=(1024, 512, 64))
    v.update(kw)
    return (ctypes.c_int64 * 18)(v["B"], v["H"], v["Hk"], v["Nq"], v["Nk"], v["D"], v["dtype"],
                                 v["kind"], v["ms"], *v["q"], *v["k"], *v["v"])


@pytest.mark.parametrize("kw,match", [
    (dict(D=60), "bad shape"), (dict(D=136), "bad shape"), (dict(D=0), "bad shape"),
    (dict(Nq=0), "bad shape"), (dict(Nk=0), "bad shape"), (dict(H=3), "bad shape"),
    (dict(Nq=1 << 31), "too many"), (dict(k=(1024, 512, 60)), "strides"),
    (dict(q=(512, -256, 64)), "strides"), (dict(k=(1024, 512, 1 << 23)), "stride too large"),
    (dict(dtype=2), "dtype"), (dict(kind=3), "bad mask"), (dict(kind=1), "disagree"),
])
def test_c_abi_cross_attention_shapes(kw, match):
    from openfold3_triangle_kernel_amd import _native

    with pytest.raises(RuntimeError, match=match):
        _native.call("tpf_xattn_forward", 16, 16, 16, None, 16, None, 16, 1 << 30, _shape(**kw), 0.125,
                     None)
    if match != "disagree":
        assert _native.query("tpf_xattn_forward_workspace_bytes", _shape(**kw)) == -1


def test_c_abi_arguments():
    from openfold3_triangle_kernel_amd import _native

    def refused(match, name, *args):
        with pytest.raises(RuntimeError, match=match):
            _native.call(name, *args)

    s, g = _shape(), (ctypes.c_int64 * 9)(512, 256, 64, 1024, 512, 64, 1024, 512, 64)
    refused("null pointer", "tpf_xattn_forward", None, 16, 16, None, 16, None, 16, 0, s, 0.1, None)
    refused("16 bytes", "tpf_xattn_forward", 8, 16, 16, None, 16, None, 16, 0, s, 0.1, None)
    refused("scale", "tpf_xattn_forward", 16, 16, 16, None, 16, None, 16, 0, s, 0.0, None)
    refused("workspace", "tpf_xattn_forward", 16, 16, 16, None, 16, None, 16, 8, _shape(Nk=4096), 0.1,
            None)
    refused("workspace", "tpf_xattn_backward_bf16", *([16] * 3), None, *([16] * 7), 8, s, g, 0.1, None)
    refused("BF16 only", "tpf_xattn_backward_bf16", *([16] * 3), None, *([16] * 7), 1 << 20,
            _shape(dtype=1), g, 0.1, None)
    bad = (ctypes.c_int64 * 9)(512, 256, 63, 1024, 512, 64, 1024, 512, 64)
    refused("gradient strides", "tpf_xattn_backward_bf16", *([16] * 3), None, *([16] * 7), 1 << 20, s,
            bad, 0.1, None)
    refused("bad shape", "tpf_norm_forward", 16, 8, 0, 8, 0, None, None, 0, 1e-5, 16, None, None, None,
            None, None)
    refused("unknown type", "tpf_norm_forward", 16, 8, 4, 8, 3, None, None, 0, 1e-5, 16, None, None,
            None, None, None)
    refused("both given or both null", "tpf_norm_forward", 16, 8, 4, 8, 0, None, None, 0, 1e-5, 16,
            None, None, 16, None, None)
    refused("means or the codes", "tpf_norm_backward", 16, None, 8, None, None, None, 16, 4, 8, 0, None,
            0, 16, 8, None, None, None, 0, None)
    refused("workspace", "tpf_norm_backward", 16, 16, 8, None, None, 16, 16, 4, 8, 0, None, 0, 16, 8,
            16, None, 16, 4, None)
    refused("8 bytes", "tpf_act8_pack", 16, 8, 4, 8, 0, 12, 16, None)
    refused("null pointer", "tpf_act8_unpack", None, 16, 4, 8, 16, 8, 0, None)
    refused("bad shape", "tpf_wgrad_act8", 16, 12, 16, 16, 4, 12, 8, 16, 0, 16, 0, None)
    refused("BF16 or FP32", "tpf_wgrad_act8", 16, 16, 16, 16, 4, 16, 8, 16, 1, 16, 0, None)
    refused("workspace", "tpf_wgrad_act8", 16, 16, 16, 16, 1 << 16, 16, 8, 16, 0, 16, 4, None)
    refused("bad shape", "tpf_row_gemm_bf16", 16, 8, 16, 1, 16, 0, 8, 8, None)


def test_block_runs_its_formulas_on_the_cpu():
    torch.manual_seed(0)
    block = CrossAttention(24, 40, 8, 4, no_kv_heads=2).double()
    x = torch.randn(2, 5, 24, dtype=torch.float64, requires_grad=True)
    kv = torch.randn(2, 7, 40, dtype=torch.float64)
    mask = torch.ones(2, 7, dtype=torch.bool)
    mask[0, 4:] = False
    mask[1] = False
    before = stock_invocation_count()
    out = block(x, kv, mask)
    assert stock_invocation_count() == before + 2  # the states' projection and the call
    assert out.shape == x.shape and not out[1].any()  # no state: nothing attended
    s = torch.nn.functional.layer_norm(kv[:, :4].float(), (40,), block.layer_norm_kv.weight.float(),
                                       block.layer_norm_kv.bias.float()).double()
    q = torch.nn.functional.layer_norm(x.float(), (24,), block.layer_norm_q.weight.float(),
                                       block.layer_norm_q.bias.float()).double()
    heads = lambda t, h: t.reshape(2, -1, h, 8).transpose(1, 2)  # noqa: E731
    k, v = (heads(m(s), 2).repeat_interleave(2, 1) for m in (block.linear_k, block.linear_v))
    p = torch.softmax(heads(block.linear_q(q), 4) @ k.transpose(-1, -2) / math.sqrt(8), -1)
    want = (p @ v).transpose(1, 2).reshape(2, 5, 32) * torch.sigmoid(block.linear_g(q))
    # The norms and the attention run in FP32 here.
    assert (out[0] - block.linear_o(want)[0]).abs().max() <= 1e-5
    states = block.project_states(kv)
    assert torch.equal(block(x, key_mask=mask, states=states), out)
    out.sum().backward()
    assert torch.isfinite(x.grad).all() and not x.grad[1].any()
    with pytest.raises(ValueError, match="either kv or states"):
        block(x)
    set_turbopairformer_strict(True)
    try:
        with pytest.raises(RuntimeError, match="strict"):
            block(x, kv)
    finally:
        set_turbopairformer_strict(False)
    for bad in (dict(no_heads=3, no_kv_heads=2), dict(no_heads=2, activation_save="int4")):
        with pytest.raises(ValueError):
            CrossAttention(8, 8, 8, **bad)


@pytest.mark.parametrize("Nq,Nk", [(3, 0), (0, 5), (0, 0)])
def test_block_of_empty_axes_on_the_cpu(Nq, Nk):
    block = CrossAttention(16, 24, 8, 4, no_kv_heads=2)
    x, kv = torch.randn(2, Nq, 16, requires_grad=True), torch.randn(2, Nk, 24, requires_grad=True)
    for mask in (None, torch.ones(2, Nk, dtype=torch.bool), torch.zeros(2, Nk)):
        out = block(x, kv, mask)
        assert out.shape == x.shape and not out.any()  # no state: nothing attended
        for g in torch.autograd.grad(out, [x, kv, *block.parameters()], torch.ones_like(out)):
            assert not g.any()


def test_c_abi_shadow_arguments():
    from openfold3_triangle_kernel_amd import _native

    s, g = _shape(), (ctypes.c_int64 * 9)(512, 256, 64, 1024, 512, 64, 1024, 512, 64)
    for match, args in (("null pointer", (16, 16, 16, None, 16, None, 16, 16, 0, s, 0.1, None)),
                        ("null pointer", (16, 16, 16, None, 16, 16, None, 16, 0, s, 0.1, None)),
                        ("16 bytes", (16, 16, 16, None, 16, 16, 8, 16, 0, s, 0.1, None)),
                        ("BF16 only", (16, 16, 16, None, 16, 16, 16, 16, 0, _shape(dtype=1), 0.1, None))):
        with pytest.raises(RuntimeError, match=match):
            _native.call("tpf_xattn_forward_shadow_bf16", *args)
    for match, residual in (("null pointer", None), ("16 bytes", 8), ("workspace", 16)):
        with pytest.raises(RuntimeError, match=match):
            _native.call("tpf_xattn_backward_shadow_bf16", 16, 16, 16, None, 16, residual, *([16] * 6), 8,
                         s, g, 0.1, None)


def test_nan_is_honoured_where_it_is_answered_for():
    """No source whose kernels carry NaN to their results is built as if there were none."""
    from openfold3_triangle_kernel_amd.build import FILE_FLAGS

    assert {name for name, flags in FILE_FLAGS.items() if any("nan" in f for f in flags)} <= {"attention.hip"}


def test_block_takes_masks_in_64_bits():
    """Finite values past the 32-bit range leave a state live, as in the kernels."""
    torch.manual_seed(0)
    block = CrossAttention(16, 24, 8, 4)
    x, kv = torch.randn(2, 3, 16), torch.randn(2, 5, 24)
    mask = torch.zeros(2, 5, dtype=torch.float64)
    mask[0, 2], mask[1] = torch.finfo(torch.float64).max, torch.finfo(torch.float64).min
    narrow = mask.clamp(torch.finfo(torch.float32).min, torch.finfo(torch.float32).max).float()
    out = block(x, kv, mask)
    assert torch.equal(out, block(x, kv, narrow)) and torch.isfinite(out).all() and out[1].any()


def test_sizes_that_a_launch_does_not_hold():
    """A launch has less than 2^32 threads: more workgroups are refused, of the backward's
    too before the forward."""
    from openfold3_triangle_kernel_amd import _native
    from openfold3_triangle_kernel_amd.cross_attention import _workspace_bytes

    most = (1 << 24) - 8
    one = dict(H=1, Hk=1, D=8, q=(8, 8, 8), k=(8, 8, 8), v=(8, 8, 8))
    for kw, forward, backward in ((dict(B=most, Nq=1, Nk=1), True, True),
                                  (dict(B=most + 1, Nq=1, Nk=1), False, False),
                                  (dict(B=most // 2, Nq=256, Nk=1), False, False),
                                  (dict(B=most // 8, Nq=64, Nk=1024), True, True),
                                  (dict(B=most // 8, Nq=64, Nk=1025), True, False)):
        shape = _shape(**one, **kw)
        for ok, name in ((forward, "tpf_xattn_forward_workspace_bytes"),
                         (backward, "tpf_xattn_backward_workspace_bytes")):
            assert (_native.query(name, shape) >= 0) == ok, (kw, name)
        for ok, grad in ((forward, False), (backward, True)):
            if ok:
                assert _workspace_bytes(shape, grad) >= 0
            else:
                with pytest.raises(ValueError, match="too many"):
                    _workspace_bytes(shape, grad)
    with pytest.raises(RuntimeError, match="too many values"):
        _native.call("tpf_act8_pack", 16, 32, 1 << 31, 32, 0, 16, 16, None)


def test_block_formulas_of_infinite_scores():
    """In the PyTorch route as in the kernels: no weight for a score of -inf, NaN for a row
    that has only such, 0 for a row without a state."""
    from openfold3_triangle_kernel_amd.cross_block import _stock_cross_attention

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 2, n, 8, generator=g) for n in (3, 5, 5))
    q[..., 0], k[..., 0] = q[..., 0].abs() + 0.5, -k[..., 0].abs() - 0.5
    for mask in (None, torch.ones(2, 5, dtype=torch.bool), torch.zeros(2, 5)):
        ks = k.clone()
        ks[:, :, 2:, 0] = float("-inf")
        part = _stock_cross_attention(q, k[:, :, :2], v[:, :, :2], None)
        assert (_stock_cross_attention(q, ks, v, mask) - part).abs().max() <= 1e-6
        ks[..., 0] = float("-inf")
        assert _stock_cross_attention(q, ks, v, mask).isnan().all()
    assert not _stock_cross_attention(q, ks, v, torch.zeros(2, 5, dtype=torch.bool)).any()


@pytest.mark.parametrize("shape,strides,read", [
    ((2, 4, 100, 64), (1 << 24, 6400, 64, 1), True),  # sequences far apart
    ((2, 4, 100, 64), (64, 1 << 24, 256, 1), True),
    ((2, 1, 100, 64), (1 << 24, 3, 64, 1), True),  # an axis of one entry
    ((1, 1, 1, 64), (1, 3, 1 << 24, 1), True),
    ((1, 4, 1, 64), (1, 64, (1 << 23) + 1, 1), True),
    ((2, 4, 100, 64), (1 << 30, 64, (1 << 23) - 8, 1), True),
    ((2, 4, 100, 64), (1 << 30, 64, 1 << 23, 1), False),
    ((2, 4, 100, 64), (25600 + 4, 6400, 64, 1), False),
    ((2, 4, 100, 64), (51200, 12800, 128, 2), False),
])
def test_cross_attention_reads_operands_in_place(shape, strides, read):
    from openfold3_triangle_kernel_amd.cross_attention import _operand

    t = torch.empty(1 << 32, dtype=torch.bfloat16, device="meta").as_strided(shape, strides)
    assert (_operand(t) is t) == read

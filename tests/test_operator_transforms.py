"""Forward-mode derivatives, function transforms and traces of the operators next to the
pair stack: the native calls are hidden from torch, so what it cannot follow is refused
or recorded as a node, with and without gradients, and never answered without it."""

import pytest
import torch
from torch.autograd import forward_ad

from openfold3_triangle_kernel_amd import (
    _native,
    activations,
    compress_activation,
    cross_attention,
    decompress_activation,
    layer_norm,
    linear,
)

# The module of that name is hidden behind the function.
_cross = __import__("sys").modules["openfold3_triangle_kernel_amd.cross_attention"]


def _operands(device="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    draw = lambda *shape: torch.randn(*shape, generator=g).bfloat16().to(device)  # noqa: E731
    return {"attend": (draw(2, 4, 70, 64), draw(2, 2, 90, 64), draw(2, 2, 90, 64), draw(2, 90)),
            "attend_padded": (draw(2, 4, 3, 20), draw(2, 2, 9, 20), draw(2, 2, 9, 20)),
            "norm": (draw(30, 64), draw(64), draw(64)), "norm_int8": (draw(30, 64), draw(64), draw(64)),
            "linear": (draw(30, 64), draw(16, 64))}


_CALLS = {"attend": lambda q, k, v, m: cross_attention(q, k, v, m),
          "attend_padded": lambda q, k, v: cross_attention(q, k, v),
          "norm": lambda x, w, b: layer_norm(x, w, b),
          "norm_int8": lambda x, w, b: layer_norm(x, w, b, save="int8"), "linear": linear}


@pytest.fixture
def fake(monkeypatch):
    """The facades on host tensors, the native calls recorded instead of made."""
    calls = []
    monkeypatch.setattr(_native, "call", lambda name, *args: calls.append(name))
    monkeypatch.setattr(_native, "query", lambda name, *args: 0)
    for module in (_cross, activations):
        monkeypatch.setattr(module, "_device_supported", lambda t: (True, ""))
    return calls


def _refuses_tangents(device):
    for name, operands in _operands(device).items():
        for i in range(len(operands)):
            for grad in (False, True):
                with forward_ad.dual_level():
                    ops = [t.clone() for t in operands]
                    if grad:
                        ops[0].requires_grad_(True)
                    ops[i] = forward_ad.make_dual(ops[i], torch.ones_like(ops[i]))
                    with pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
                        _CALLS[name](*ops)
                    with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError),
                                                        match="forward|jvp"):
                        _CALLS[name](*ops)


def test_forward_mode_is_refused(fake):
    _refuses_tangents("cpu")


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu(gpu):
    _refuses_tangents(gpu)


def test_function_transforms_are_refused(fake):
    for name, operands in _operands().items():
        with pytest.raises(RuntimeError, match="functorch|vmap|data pointer"):
            torch.vmap(lambda t: _CALLS[name](t, *operands[1:]))(operands[0][None].repeat(3, *[1] * operands[0].ndim))
        with pytest.raises((RuntimeError, NotImplementedError), match="functorch|jvp|forward|data pointer"):
            torch.func.jvp(lambda t: _CALLS[name](t, *operands[1:]), operands[:1], operands[:1])


def test_traces_hold_the_operators(fake):
    for name, operands in _operands().items():
        for grad in (False, True):
            ops = tuple(t.clone().requires_grad_(grad and i == 0) for i, t in enumerate(operands))
            graph = str(torch.jit.trace(_CALLS[name], ops, check_trace=False).graph)
            assert "^_" in graph, f"{name}: no node for the operator in\n{graph}"


@pytest.mark.gpu
def test_traces_compute(gpu):
    """A traced function gives what the call gives on other operands."""
    first, second = _operands(gpu, 1), _operands(gpu, 2)
    for name, call in _CALLS.items():
        traced = torch.jit.trace(call, first[name], check_trace=False)
        want = call(*second[name])
        assert torch.equal(traced(*second[name]), want), name


def _there_and_back(x):
    return decompress_activation(compress_activation(x), torch.float32)


def test_codec_takes_values_only(fake):
    """No derivative passes through the codec, forward mode included; a trace holds it."""
    x = torch.randn(30, 64)
    with forward_ad.dual_level():
        out = _there_and_back(forward_ad.make_dual(x, torch.ones_like(x)))
        assert forward_ad.unpack_dual(out).tangent is None
    graph = str(torch.jit.trace(_there_and_back, (x,), check_trace=False).graph)
    assert graph.count("^_") == 2, graph
    with pytest.raises(RuntimeError, match="functorch|vmap|data pointer"):
        torch.vmap(_there_and_back)(x[None])


@pytest.mark.gpu
def test_traced_codec_computes(gpu):
    x, y = (torch.randn(30, 64, generator=torch.Generator().manual_seed(s)).to(gpu) for s in (1, 2))
    traced = torch.jit.trace(_there_and_back, (x,), check_trace=False)
    assert torch.equal(traced(y), _there_and_back(y)) and not torch.equal(traced(y), traced(x))

"""The cross-attention block: its operators together, as a model uses them.

Against its formulas in FP64 at the same BF16 operands.  The chain rounds to BF16
(2^-8 relative each) at the norm, the projections, the probabilities, the attention,
the gate's two factors and the output: ten roundings forward, as many again on the
way back.  Weights' gradients read 8-bit values: a uniform error of at most half a
step, the largest of a block being at least 63.75 steps, so at most 1 / (63.75 sqrt 12)
of the block's largest, which for 32 normal values is below 4 of their rms: 0.018.
"""

import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _make(gpu, save="int8", gating=True, **kw):
    from openfold3_triangle_kernel_amd import CrossAttention

    torch.manual_seed(1)
    size = dict(c_q=128, c_kv=192, c_hidden=32, no_heads=8, no_kv_heads=2)
    size.update(kw)
    block = CrossAttention(**size, gating=gating, activation_save=save)
    with torch.no_grad():
        for n, p in block.named_parameters():
            if "layer_norm" in n:
                p.add_(0.2 * torch.randn_like(p))
    return block.to(gpu)


def _formula(block, x, kv, mask):
    ln = lambda m, t: torch.nn.functional.layer_norm(t, m.normalized_shape, m.weight, m.bias, m.eps)  # noqa: E731
    xs, s = ln(block.layer_norm_q, x), ln(block.layer_norm_kv, kv)
    heads = lambda t: t.unflatten(-1, (-1, block.c_hidden)).transpose(-2, -3)  # noqa: E731
    q, k, v = heads(block.linear_q(xs)), heads(block.linear_k(s)), heads(block.linear_v(s))
    g = block.no_heads // block.no_kv_heads
    k, v = k.repeat_interleave(g, -3), v.repeat_interleave(g, -3)
    a = q @ k.transpose(-1, -2).contiguous() / math.sqrt(block.c_hidden)
    if mask is not None:
        a = a.masked_fill(~mask[..., None, None, :], float("-inf"))
    o = (torch.softmax(a, -1) @ v).transpose(-2, -3).flatten(-2)
    if block.linear_g is not None:
        o = o * torch.sigmoid(block.linear_g(xs))
    return block.linear_o(o)


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.parametrize("save", ["int8", "full"])
@pytest.mark.parametrize("gating", [True, False])
def test_block_and_gradients(gpu, save, gating):
    from openfold3_triangle_kernel_amd import stock_invocation_count

    block = _make(gpu, save, gating).bfloat16()
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 70, 128, generator=g).bfloat16().to(gpu).requires_grad_(True)
    kv = torch.randn(2, 3, 150, 192, generator=g).bfloat16().to(gpu).requires_grad_(True)
    mask = (torch.arange(150) < torch.tensor([[150, 90, 7], [33, 150, 64]])[..., None]).to(gpu)
    dout = torch.randn(2, 3, 70, 128, generator=g).bfloat16().to(gpu)
    before = stock_invocation_count()
    out = block(x, kv, mask)
    grads = torch.autograd.grad(out, [x, kv, *block.parameters()], dout)
    assert stock_invocation_count() == before
    ref = copy.deepcopy(block).double().cpu()
    xr, kr = (t.detach().double().cpu().requires_grad_(True) for t in (x, kv))
    want = _formula(ref, xr, kr, mask.cpu())
    wgrads = torch.autograd.grad(want, [xr, kr, *ref.parameters()], dout.double().cpu())
    u = 2.0 ** -8
    assert _rel(out, want) <= 10 * u
    names = ["x", "kv", *(n for n, _ in block.named_parameters())]
    for name, got, w in zip(names, grads, wgrads):
        assert _rel(got, w) <= 20 * u + (0.018 if save == "int8" else 0.0), name


def test_fp32_parameters_and_steps(gpu):
    """FP32 parameters under an optimizer: gradients in FP32, steps run."""
    block = _make(gpu)
    x = torch.randn(4, 33, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    kv = torch.randn(4, 65, 192, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    opt = torch.optim.SGD(block.parameters(), lr=1e-2)
    for _ in range(2):
        opt.zero_grad()
        block(x, kv).float().square().mean().backward()
        assert all(p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all()
                   for p in block.parameters())
        opt.step()


def test_single_tokens_from_kept_states(gpu):
    """Token by token against the kept states: the rows of the whole call, up to the
    order of the sums (few rows run on another kernel): one rounding of the attention's
    output carried through the gate and the last product."""
    block = _make(gpu).bfloat16()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 70, 128, generator=g).bfloat16().to(gpu)
    kv = torch.randn(2, 300, 192, generator=g).bfloat16().to(gpu)
    mask = (torch.arange(300) < torch.tensor([[300], [120]])).to(gpu)
    with torch.no_grad():
        whole = block(x, kv, mask)
        states = block.project_states(kv)
        assert torch.equal(block(x, key_mask=mask, states=states), whole)
        tokens = torch.cat([block(x[:, i:i + 1], key_mask=mask, states=states) for i in range(70)], 1)
    assert _rel(tokens, whole) <= 4 * 2.0 ** -8


def test_activations_kept(gpu):
    """What a training forward keeps of streams that nothing else holds: five BF16
    tensors (the norms' inputs and the projections') against five of 33/32 byte."""
    kept = {}
    x = torch.randn(4, 1024, 512, device=gpu).bfloat16().requires_grad_(True)
    for save in ("int8", "full"):
        block = _make(gpu, save, c_q=512, c_kv=512, c_hidden=64, no_heads=8, no_kv_heads=8).bfloat16()
        block(x, x.detach())  # workspaces once
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        out = block(x + 1.0, x - 1.0)
        kept[save] = torch.cuda.memory_allocated() - base
        del out
    rows = 4 * 1024 * 512
    assert kept["full"] - kept["int8"] >= rows * 5 * (2 - 33 / 32) * 0.95, kept


def test_block_captured_into_a_graph(gpu):
    block = _make(gpu).bfloat16()
    x = torch.randn(2, 40, 128, device=gpu).bfloat16()
    kv = torch.randn(2, 90, 192, device=gpu).bfloat16()
    params = list(block.parameters())

    def step():
        xs = x.detach().requires_grad_(True)
        out = block(xs, kv)
        return [out.detach(), *torch.autograd.grad(out, [xs, *params], torch.ones_like(out))]

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(2, 40, 128, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused(gpu):
    """Differentiating a gradient again raises, on the C++ host path and on Python's."""
    from openfold3_triangle_kernel_amd import cross_attention, layer_norm, linear

    def leaf(*shape):
        return torch.randn(*shape, device=gpu).bfloat16().requires_grad_(True)

    q, k, x, w = leaf(1, 2, 70, 64), leaf(1, 2, 90, 64), leaf(30, 64), leaf(16, 64)
    calls = [(lambda: cross_attention(q, k, k), q), (lambda: layer_norm(x, w[0]), x),
             (lambda: linear(x, w), x), (lambda: linear(x, w, save="full"), w),
             (lambda: cross_attention(q[..., :60], k[..., :60], k[..., :60]), k),
             (lambda: layer_norm(x[:, ::2], save="int8"), x)]
    for call, wrt in calls:
        out = call()
        g, = torch.autograd.grad(out, wrt, torch.ones_like(out), create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


@pytest.mark.parametrize("Nq,Nk", [(3, 0), (0, 5), (0, 0)])
def test_block_of_empty_axes(gpu, Nq, Nk):
    block = _make(gpu).bfloat16()
    x = torch.randn(2, Nq, 128, device=gpu).bfloat16().requires_grad_(True)
    kv = torch.randn(2, Nk, 192, device=gpu).bfloat16().requires_grad_(True)
    for mask in (None, torch.ones(2, Nk, dtype=torch.bool, device=gpu), torch.zeros(2, Nk, device=gpu)):
        out = block(x, kv, mask)
        assert out.shape == x.shape and not out.any()  # no state: nothing attended
        params = list(block.parameters())
        grads = torch.autograd.grad(out, [x, kv, *params], torch.ones_like(out), allow_unused=True)
        assert not any(g.any() for g in grads if g is not None)

"""The self-attention block: its operators together, as a model trains and serves with them.

Against its formulas in FP64 at the same BF16 operands.  The chain rounds to BF16 (2^-8
relative each) at the norm, the projections, the rotation, the probabilities, the
attention, the gate's two factors and the output: twelve roundings forward, as many again on
the way back.  Weights' gradients read 8-bit values: 0.018 (as the cross-attention block's).
"""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _make(gpu, **kw):
    from openfold3_triangle_kernel_amd import SelfAttention

    torch.manual_seed(1)
    size = dict(c_in=128, c_hidden=32, no_heads=8, no_kv_heads=2, window=30, sinks=3)
    size.update(kw)
    block = SelfAttention(**size)
    with torch.no_grad():
        for n, p in block.named_parameters():
            if "norm" in n:
                p.add_(0.2 * torch.randn_like(p))
    return block.to(gpu)


def _formula(block, x, mask):
    """On the CPU in the operands' type (64 bits), apart from the block's own route."""
    h = torch.nn.functional.layer_norm(x, (block.c_in,), block.layer_norm.weight, block.layer_norm.bias, block.eps)
    heads = lambda m: m(h).unflatten(-1, (-1, block.c_hidden)).transpose(-2, -3)  # noqa: E731
    q, k, v = heads(block.linear_q), heads(block.linear_k), heads(block.linear_v)
    N = x.shape[-2]
    f = block._frequencies["cpu"]
    spin = torch.polar(torch.ones(N, len(f), dtype=torch.float64), torch.arange(N).double()[:, None] * f)

    def turn(t, w):
        if w is not None:
            t = t / (t.square().mean(-1, keepdim=True) + block.eps).sqrt() * w
        n = len(f)
        if block.interleaved:
            z = torch.complex(t[..., 0:2 * n:2], t[..., 1:2 * n:2]) * spin
            turned = torch.stack((z.real, z.imag), -1).flatten(-2)
        else:
            z = torch.complex(t[..., :n], t[..., n:2 * n]) * spin
            turned = torch.cat((z.real, z.imag), -1)
        return torch.cat((turned, t[..., 2 * n:]), -1)

    q, k = turn(q, block.norm_q), turn(k, block.norm_k)
    g = block.no_heads // block.no_kv_heads
    k, v = k.repeat_interleave(g, -3), v.repeat_interleave(g, -3)
    far = torch.arange(N)[:, None] - torch.arange(N)
    see = far >= 0
    if block.window is not None:
        see = see & ((far < block.window) | (torch.arange(N) < block.sinks))
    if mask is not None:
        see = see & mask[..., None, None, :]
    a = (q @ k.transpose(-1, -2) / block.c_hidden ** 0.5).masked_fill(~see, float("-inf"))
    p = torch.nan_to_num(torch.softmax(a, -1))
    o = (p @ v).transpose(-2, -3).flatten(-2)
    if block.linear_g is not None:
        o = o * torch.sigmoid(block.linear_g(h))
    return block.linear_o(o)


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.parametrize("kw", [dict(), dict(gating=False, activation_save="full", window=None, sinks=0),
                                dict(qk_norm=False, interleaved=True, rotary_channels=16),
                                dict(c_hidden=64, no_kv_heads=8, rotary_channels=0)], ids=str)
def test_block_and_gradients(gpu, kw):
    from openfold3_triangle_kernel_amd import stock_invocation_count

    block = _make(gpu, **kw).bfloat16()
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 2, 150, 128, generator=g).bfloat16().to(gpu).requires_grad_(True)
    mask = (torch.arange(150) < torch.tensor([[150, 90], [33, 150]])[..., None]).to(gpu)
    dout = torch.randn(2, 2, 150, 128, generator=g).bfloat16().to(gpu)
    before = stock_invocation_count()
    out = block(x, mask)
    grads = torch.autograd.grad(out, [x, *block.parameters()], dout)
    assert stock_invocation_count() == before
    ref = copy.deepcopy(block).double().cpu()
    xr = x.detach().double().cpu().requires_grad_(True)
    want = _formula(ref, xr, mask.cpu())
    wgrads = torch.autograd.grad(want, [xr, *ref.parameters()], dout.double().cpu())
    u = 2.0 ** -8
    assert _rel(out, want) <= 12 * u
    for name, got, w in zip(["x", *(n for n, _ in block.named_parameters())], grads, wgrads):
        assert _rel(got, w) <= 24 * u + 0.018, name


@pytest.mark.parametrize("kw", [dict(), dict(window=None, interleaved=True)], ids=str)
def test_prompts_and_tokens_through_a_cache(gpu, kw):
    """Two sequences in chunks and single tokens through the cache, in batches with a row of
    no sequence: the rows of the whole call, up to the order of the sums and one rounding of
    the attention's output carried on."""
    block = _make(gpu, **kw).bfloat16()
    g = torch.Generator().manual_seed(3)
    total = (90, 61)
    xs = [torch.randn(n, 128, generator=g).bfloat16().to(gpu) for n in total]
    with torch.no_grad():
        whole = [block(x) for x in xs]
    cache = block.new_cache(14, 16)
    tables = torch.randperm(14, generator=g)[:12].view(2, 6).int().to(gpu)
    at, got = [0, 0], [[], []]
    for news in ((40, 1), (1, 30), (1, 1), (1, 1), (47, 28)):
        starts = torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device=gpu)
        rows = [x[a:a + n] for x, a, n in zip(xs, at, news)]
        at = [a + n for a, n in zip(at, news)]
        lengths = torch.tensor(at, dtype=torch.int32, device=gpu)
        out = block.step(torch.cat(rows + [xs[0][:1]]), cache, tables, starts, lengths)
        got[0].append(out[:news[0]])
        got[1].append(out[news[0]:sum(news)])
        assert not out[sum(news):].any()
    assert at == list(total)
    for o, w in zip(got, whole):
        assert _rel(torch.cat(o), w) <= 4 * 2.0 ** -8


def test_step_replays(gpu):
    """A captured step serves the next tokens, its tables and lengths changed in place."""
    block = _make(gpu).bfloat16()
    g = torch.Generator().manual_seed(4)
    xs = torch.randn(40, 2, 128, generator=g).bfloat16().to(gpu)
    tables = torch.arange(10, dtype=torch.int32, device=gpu).view(2, 5)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    runs = []
    for captured in (False, True):
        cache = block.new_cache(10, 8)
        x, lengths = xs[0].clone(), torch.ones(2, dtype=torch.int32, device=gpu)
        block.step(x, cache, tables, starts, lengths)  # workspaces once
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                held = block.step(x, cache, tables, starts, lengths)
        outs = []
        for i in range(40):
            x.copy_(xs[i])
            lengths.fill_(i + 1)
            if captured:
                graph.replay()
                outs.append(held.clone())
            else:
                outs.append(block.step(x, cache, tables, starts, lengths))
        runs.append(torch.stack(outs))
    assert torch.equal(*runs)


def test_fp32_parameters_and_steps(gpu):
    """FP32 parameters under an optimizer: gradients in FP32, steps run."""
    block = _make(gpu)
    x = torch.randn(4, 65, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    opt = torch.optim.SGD(block.parameters(), lr=1e-2)
    for _ in range(2):
        opt.zero_grad()
        block(x).float().square().mean().backward()
        assert all(p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all()
                   for p in block.parameters())
        opt.step()


def test_stock_route_agrees(gpu):
    """FP32 activations take the PyTorch route: the same rows to the kernels' roundings."""
    from openfold3_triangle_kernel_amd import stock_invocation_count

    block = _make(gpu).bfloat16()
    x = torch.randn(2, 80, 128, generator=torch.Generator().manual_seed(5)).bfloat16().to(gpu)
    mask = torch.ones(2, 80, dtype=torch.bool, device=gpu)
    mask[1, :20] = False
    with torch.no_grad():
        want = block(x, mask)
        before = stock_invocation_count()
        got = copy.deepcopy(block).float()(x.float(), mask)
        assert stock_invocation_count() == before + 1
    assert _rel(want, got) <= 12 * 2.0 ** -8
    with pytest.raises(ValueError, match="BF16"):
        block.step(x[0].float(), None, None, None, None)


def test_trains_after_inference_mode(gpu):
    block = _make(gpu)
    x = torch.randn(1, 40, 128, device=gpu).bfloat16()
    with torch.inference_mode():
        want = block(x)
    out = block(x)
    out.float().sum().backward()
    assert torch.equal(out, want) and all(p.grad is not None for p in block.parameters())


def test_block_without_tokens(gpu):
    block = _make(gpu)
    x = torch.zeros(2, 0, 128, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    out = block(x)
    out.sum().backward()
    assert out.shape == x.shape and x.grad.shape == x.shape
    cache = block.new_cache(2, 8, gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    out = block.step(x.detach()[0], cache, none.reshape(0, 1), none.new_zeros(1), none)
    assert out.shape == (0, 128)
    out = block.step(torch.randn(3, 128, device=gpu).bfloat16(), cache, none.reshape(0, 1), none.new_zeros(1), none)
    assert not out.any() and not cache.k.any()  # tokens of no sequence

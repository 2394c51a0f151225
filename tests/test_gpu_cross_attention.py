"""Cross attention against the formulas in 64 bits.

Tolerances count roundings.  With u = finfo(type).eps / 2: the probabilities enter
the second product rounded (u each), outputs are rounded once (u), and the scores
carry D + 4 roundings of 32 bits, ds = (D + 4) 2^-24 scale sum |q||k|, which a
softmax turns into a relative error of at most 2 ds (numerator and sum); the
exponential and the sums add 2^-20 and (Nk / 32 + 64) 2^-24.  FP16 probabilities
below 2^-14 are subnormal: 2^-25 each, the largest being at least 1.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _make(dev, B, H, Hk, Nq, Nk, D, dtype=torch.bfloat16, layout="head", seed=0, qscale=1.5):
    g = torch.Generator().manual_seed(seed)

    def heads(h, n, scale=1.0):
        if layout == "seq":
            t = torch.randn(B, n, h, D, generator=g).mul(scale).to(dtype).to(dev)
            return t.transpose(1, 2)
        if layout == "fused":  # a slice of a wider projection
            t = torch.randn(B, n, h, 2 * D, generator=g).mul(scale).to(dtype).to(dev)
            return t[..., D:].transpose(1, 2)
        return torch.randn(B, h, n, D, generator=g).mul(scale).to(dtype).to(dev)

    return heads(H, Nq, qscale), heads(Hk, Nk), heads(Hk, Nk)


def _mask(dev, kind, B, Nk, seed=0):
    g = torch.Generator().manual_seed(100 + seed)
    if kind == "none":
        return None
    if kind == "tail":
        live = Nk - torch.randint(0, Nk // 2 + 1, (B, 1), generator=g)
        return (torch.arange(Nk) < live).to(dev)
    if kind == "random":
        return (torch.rand(B, Nk, generator=g) < 0.4).to(dev)
    if kind == "empty":
        m = torch.rand(B, Nk, generator=g) < 0.7
        m[0] = False
        return m.to(dev)
    if kind == "add":
        m = torch.randn(B, Nk, generator=g)
        m[torch.rand(B, Nk, generator=g) < 0.3] = float("-inf")
        return m.to(dev)
    if kind == "add_empty":
        m = torch.randn(B, Nk, generator=g)
        m[0] = float("-inf")
        return m.to(dev)
    raise AssertionError(kind)


def _reference(q, k, v, mask, scale, dout=None):
    """Outputs, their error bounds, and the same of the gradients, in 64 bits."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1:3]
    G = H // Hk
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    live = torch.ones(B, Nk, dtype=torch.bool)
    add = torch.zeros(B, Nk, dtype=torch.float64)
    if mask is not None:
        mask = mask.cpu()
        if mask.dtype == torch.bool:
            live = mask.expand(B, Nk)
        else:
            add = mask.double().expand(B, Nk)
            live = ~torch.isneginf(add)
    k = torch.where(live[:, None, :, None], k, 0.0)
    v = torch.where(live[:, None, :, None], v, 0.0)
    ke, ve = (t.repeat_interleave(G, 1) for t in (k, v))
    s = scale * q @ ke.transpose(-1, -2) + torch.where(live, add, 0.0)[:, None, None, :]
    s = s.masked_fill(~live[:, None, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ ve
    ds_ = (D + 4) * 2.0 ** -24 * (scale * (q.abs() @ ke.abs().transpose(-1, -2))).amax(-1, keepdim=True)
    ds_ = ds_ + 2.0 ** -22 * torch.where(live, add, 0.0).abs().amax(-1)[:, None, None, None]
    rel = 2 * ds_ + 2.0 ** -20 + (Nk / 32 + 64) * 2.0 ** -24
    eo = u * o.abs() + (u + rel) * (p @ ve.abs()) * (1 + u) + sub * ve.abs().sum(-2, keepdim=True) + 2 * sub
    outs, errs = [o.transpose(1, 2)], [eo.transpose(1, 2)]
    if dout is None:
        return outs, errs
    do = dout.detach().double().cpu().transpose(1, 2)
    dp = do @ ve.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    edelta = (do.abs() * eo).sum(-1, keepdim=True) + D * 2.0 ** -24 * (do.abs() * o.abs()).sum(-1, keepdim=True)
    edp = (D + 4) * 2.0 ** -24 * (do.abs() @ ve.abs().transpose(-1, -2))
    ds = p * (dp - delta)
    eds = (u + rel) * ds.abs() * (1 + u) + p * (edelta + edp) * (1 + u + rel)
    sums = (G * Nq / 16 + Nk / 16 + 64) * 2.0 ** -24

    def group(t):  # sums over the query heads of a kv head
        return t.reshape(B, Hk, G, Nk, D).sum(2)

    dq, dk = scale * ds @ ke, group(scale * ds.transpose(-1, -2) @ q)
    dv = group(p.transpose(-1, -2) @ do)
    edq = u * dq.abs() + scale * ((eds + sums * ds.abs()) @ ke.abs()) * (1 + u)
    edk = u * dk.abs() + group(scale * (eds + sums * ds.abs()).transpose(-1, -2) @ q.abs()) * (1 + u)
    edv = u * dv.abs() + group(((u + rel + sums) * p).transpose(-1, -2) @ do.abs()) * (1 + u)
    return outs + [dq, dk, dv], errs + [edq, edk, edv]


def _check(got, want, tol, names=("out", "dq", "dk", "dv")):
    for g, w, t, name in zip(got, want, tol, names):
        g = g.detach().double().cpu()
        assert g.shape == w.shape, name
        over = ((g - w).abs() - t - 1e-30).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"


FORWARD = [
    # B, H, Hk, Nq, Nk, D, type, layout, mask
    (1, 1, 1, 1, 1, 8, "bf16", "head", "none"),
    (2, 8, 8, 1, 77, 64, "bf16", "head", "none"),
    (3, 8, 2, 1, 1000, 128, "bf16", "seq", "tail"),
    (2, 8, 1, 1, 4099, 128, "fp16", "fused", "random"),
    (2, 32, 1, 2, 513, 96, "bf16", "head", "empty"),
    (1, 4, 4, 65, 33, 32, "bf16", "head", "none"),
    (2, 4, 2, 100, 200, 64, "fp16", "seq", "add"),
    (2, 2, 1, 129, 64, 40, "bf16", "fused", "random"),
    (1, 3, 3, 300, 129, 80, "bf16", "seq", "none"),
    (2, 6, 2, 257, 500, 128, "bf16", "head", "add_empty"),
    (2, 2, 2, 70, 63, 20, "bf16", "head", "tail"),
    (1, 1, 1, 64, 2500, 72, "fp16", "head", "none"),
    (1, 2, 1, 130, 6000, 128, "bf16", "head", "tail"),
    (1, 2, 2, 1, 1100, 64, "bf16", "seq", "random"),  # a few splits
    (1, 2, 2, 100, 650, 96, "bf16", "head", "empty"),
    (1, 1, 1, 1, 70001, 32, "bf16", "head", "none"),  # as many as there may be
    (1, 8, 1, 5, 1500, 128, "fp16", "head", "add"),
    (1, 64, 64, 300, 70, 64, "bf16", "head", "tail"),  # 256 rows a workgroup needs 512 of them
    (4, 64, 64, 513, 65, 48, "fp16", "seq", "random"),
    (8, 64, 64, 260, 70, 32, "bf16", "seq", "add"),
]
_T = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("case", FORWARD, ids=str)
def test_forward(gpu, case):
    from openfold3_triangle_kernel_amd import cross_attention

    B, H, Hk, Nq, Nk, D, t, layout, mk = case
    q, k, v = _make(gpu, B, H, Hk, Nq, Nk, D, _T[t], layout)
    mask = _mask(gpu, mk, B, Nk)
    want, tol = _reference(q, k, v, mask, 1 / math.sqrt(D))
    with torch.no_grad():
        out = cross_attention(q, k, v, mask)
    assert out.shape == (B, Nq, H, D) and out.is_contiguous()
    _check([out], want, tol)
    if mk in ("empty", "add_empty"):
        assert torch.equal(out[0], torch.zeros_like(out[0]))


BACKWARD = [
    # B, H, Hk, Nq, Nk, D, layout, mask
    (1, 1, 1, 1, 1, 8, "head", "none"),
    (2, 4, 2, 1, 65, 64, "seq", "tail"),
    (2, 4, 4, 33, 100, 32, "head", "random"),
    (2, 8, 2, 129, 257, 64, "fused", "empty"),
    (3, 4, 1, 67, 190, 80, "seq", "add_empty"),
    (1, 2, 2, 130, 64, 96, "head", "none"),
    (2, 4, 2, 200, 333, 128, "seq", "tail"),
    (1, 8, 1, 300, 1500, 128, "head", "add"),
    (1, 2, 1, 16, 3001, 40, "head", "random"),
    (1, 1, 1, 1500, 65, 20, "seq", "none"),
]


@pytest.mark.parametrize("case", BACKWARD, ids=str)
def test_backward(gpu, case):
    from openfold3_triangle_kernel_amd import cross_attention

    B, H, Hk, Nq, Nk, D, layout, mk = case
    q, k, v = (t.requires_grad_(True) for t in _make(gpu, B, H, Hk, Nq, Nk, D, layout=layout, seed=3))
    mask = _mask(gpu, mk, B, Nk, 3)
    dout = torch.randn(B, Nq, H, D, generator=torch.Generator().manual_seed(9)).bfloat16().to(gpu)
    want, tol = _reference(q, k, v, mask, 1 / math.sqrt(D), dout)
    out = cross_attention(q, k, v, mask)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    _check([out, *grads], want, tol)
    again = torch.autograd.grad(cross_attention(q, k, v, mask), (q, k, v), dout)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)


def test_gradients_against_differences(gpu):
    """Directional differences of the 64-bit formula at the BF16 operands: the
    gradient's own roundings (2^-9 relative, a few of them) bound the deviation."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = (t.requires_grad_(True) for t in _make(gpu, 1, 2, 1, 40, 50, 64, seed=5))
    mask = _mask(gpu, "tail", 1, 50, 5)
    dout = torch.randn(1, 40, 2, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    grads = torch.autograd.grad(cross_attention(q, k, v, mask), (q, k, v), dout)
    base = [t.detach().double().cpu() for t in (q, k, v)]

    def loss(ops):
        return (_reference(*ops, mask, 1 / 8.0)[0][0] * dout.double().cpu()).sum().item()

    for n in range(3):
        g = grads[n].double().cpu()
        step = g / g.norm()
        h = 1e-5
        ops = [list(base), list(base)]
        ops[0][n], ops[1][n] = base[n] + h * step, base[n] - h * step
        slope = (loss(ops[0]) - loss(ops[1])) / (2 * h)
        assert abs(slope - g.norm().item()) <= 2.0 ** -7 * g.norm().item()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("Nq,D", [(1, 128), (70, 64), (200, 128)])
def test_dropped_states_are_never_used(gpu, bad, Nq, D):
    """Whatever K and V hold at dropped states, results are those of zeros there."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 2, 4, 2, Nq, 150, D, seed=7)
    for mask in (_mask(gpu, "random", 2, 150, 7), _mask(gpu, "add_empty", 2, 150, 7)):
        dead = (~mask if mask.dtype == torch.bool else torch.isneginf(mask))[:, None, :, None]
        runs = []
        for fill in (0.0, bad):
            ops = [t.detach().clone().requires_grad_(True)
                   for t in (q, k.masked_fill(dead, fill), v.masked_fill(dead, fill))]
            out = cross_attention(*ops, mask)
            runs.append([out, *torch.autograd.grad(out, ops, torch.ones_like(out))])
        for a, b in zip(*runs):
            assert torch.isfinite(b).all() and torch.equal(a, b)
        assert not runs[1][2][dead.expand_as(k)].any() and not runs[1][3][dead.expand_as(v)].any()


@pytest.mark.parametrize("Nq,Nk,D", [(1, 1, 64), (1, 300, 64), (3, 1000, 128), (130, 700, 64),
                                     (300, 200, 96), (512, 1024, 128)])
def test_nan_in_live_places_is_not_lost(gpu, Nq, Nk, D):
    """NaN in q, k, v or an additive mask reaches all that the formula makes of it, and
    nothing else: a row, a kv head, a channel of a kv head, a batch entry."""
    from openfold3_triangle_kernel_amd import cross_attention

    nan = float("nan")
    ops = _make(gpu, 2, 4, 2, Nq, Nk, D, seed=9)
    zero = torch.zeros(2, Nk, device=gpu)

    def run(q, k, v, mask):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = cross_attention(*leaves, mask)
        return (out, *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    clean = run(*ops, zero)
    for what in range(4):
        q, k, v, mask = (t.detach().clone() for t in (*ops, zero))
        hit = torch.zeros(2, Nq, 4, D, dtype=torch.bool, device=gpu)  # of the output
        if what == 0:
            q[0, 1, Nq // 2, 5] = nan
            hit[0, Nq // 2, 1] = True
        elif what == 1:
            k[0, 1, Nk // 2, 5] = nan
            hit[0, :, 2:] = True
        elif what == 2:
            v[0, 1, Nk // 2, 5] = nan
            hit[0, :, 2:, 5] = True
        else:
            mask[0, Nk // 2] = nan
            hit[0] = True
        out, dq, dk, dv = run(q, k, v, mask)
        assert torch.equal(out.isnan(), hit)
        assert torch.equal(out[~hit], clean[0][~hit])
        if what == 3:
            for g, c in zip((dq, dk, dv), clean[1:]):
                assert g[0].isnan().all() and torch.equal(g[1], c[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Nq", [1, 100])
def test_lowest_finite_mask(gpu, dtype, Nq):
    """A row whose states all carry the type's lowest value has live states: the
    scores vanish beside it, the row is their mean (as in 32-bit arithmetic) for
    the 32-bit range, and it drops out beside states without it."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 2, 2, 2, Nq, 130, 64, seed=8)
    low = torch.finfo(dtype).min
    mask = torch.zeros(2, 130, dtype=dtype, device=gpu)
    mask[0, 40:] = low
    mask[1] = low
    with torch.no_grad():
        out = cross_attention(q, k, v, mask)
        part = cross_attention(q[:1], k[:1, :, :40], v[:1, :, :40])
    assert torch.equal(out[:1], part) or (out[:1].float() - part.float()).abs().max() <= 2.0 ** -7
    if dtype != torch.float16:
        mean = v[1].double().mean(-2)  # [H, D]
        u = 2.0 ** -8
        bound = 2 * u * v[1].double().abs().mean(-2) + 1e-6
        assert ((out[1].double() - mean).abs() <= bound).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("Nq", [1, 100])
def test_highest_finite_mask(gpu, Nq):
    """States with the type's highest value outweigh all others: the row is their mean
    (the scores vanish beside it), and the others' gradients are 0."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = (t.requires_grad_(True) for t in _make(gpu, 2, 2, 2, Nq, 130, 64, seed=8))
    mask = torch.randn(2, 130, generator=torch.Generator().manual_seed(8)).to(gpu)
    mask[0, 70:72] = mask[1, 5:7] = torch.finfo(torch.float32).max
    out = cross_attention(q, k, v, mask)
    dv, = torch.autograd.grad(out, v, torch.ones_like(out))
    for b, top in ((0, slice(70, 72)), (1, slice(5, 7))):
        pair = v[b, :, top].double()
        # p = 1 / 2 is exact, the output rounded once; dv sums Nq halves, rounded once.
        assert ((out[b].double() - pair.mean(-2)).abs() <= 2.0 ** -8 * pair.abs().sum(-2)).all()
        assert ((dv[b, :, top].double() - Nq / 2).abs() <= 2.0 ** -8 * Nq / 2).all()
        rest = torch.ones(130, dtype=torch.bool, device=gpu)
        rest[top] = False
        assert not dv[b][:, rest].any()


def test_masks_that_broadcast(gpu):
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 6, 2, 1, 70, 90, 32, seed=4)
    q, k, v = (t.reshape(2, 3, *t.shape[1:]) for t in (q, k, v))
    with torch.no_grad():
        for m in (_mask(gpu, "random", 1, 90)[0], _mask(gpu, "random", 3, 90),
                  _mask(gpu, "random", 2, 90)[:, None], _mask(gpu, "add", 1, 90)[0].bfloat16(),
                  _mask(gpu, "random", 90, 6).t()[:3]):
            full = m.expand(2, 3, 90).contiguous()
            assert torch.equal(cross_attention(q, k, v, m), cross_attention(q, k, v, full))


def test_broadcast_and_offset_operands(gpu):
    """Expanded operands sum their gradients, storage off the 16 bytes is copied."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 1, 4, 2, 33, 70, 64, seed=6)
    dout = torch.randn(3, 33, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    ks, vs = k.clone().requires_grad_(True), v.clone().requires_grad_(True)
    q3 = q.repeat(3, 1, 1, 1)
    out = cross_attention(q3, ks.expand(3, -1, -1, -1), vs.expand(3, -1, -1, -1))
    got = torch.autograd.grad(out, (ks, vs), dout)
    k3, v3 = (t.repeat(3, 1, 1, 1).requires_grad_(True) for t in (k, v))
    out3 = cross_attention(q3, k3, v3)
    want = torch.autograd.grad(out3, (k3, v3), dout)
    assert torch.equal(out, out3)
    for g, w in zip(got, want):
        full = w.double().sum(0, keepdim=True)
        # The three terms are added in BF16: two roundings of partial sums.
        assert ((g.double() - full).abs() <= 2 * 2.0 ** -8 * w.double().abs().sum(0)).all()
    flat = torch.zeros(k.numel() + 8, device=gpu, dtype=k.dtype)
    for off in (1, 3, 4):
        shifted = flat[off:off + k.numel()].view(k.shape)
        shifted.copy_(k)
        with torch.no_grad():
            assert torch.equal(cross_attention(q, shifted, v), cross_attention(q, k, v))
    wide = torch.zeros(1, 2, 70, 67, device=gpu, dtype=k.dtype)  # odd state stride
    wide[..., :64] = k
    with torch.no_grad():
        assert torch.equal(cross_attention(q, wide[..., :64], v), cross_attention(q, k, v))


@pytest.mark.parametrize("axis", ["batch", "head", "position", "all"])
def test_gradients_of_broadcast_operands(gpu, axis):
    """Operands broadcast along any axis: the gradients are those of their copies,
    summed (in BF16, 2^-8 of the terms for each of the additions)."""
    from openfold3_triangle_kernel_amd import cross_attention

    full = {"batch": (3, 1, 1), "head": (1, 4, 1), "position": (1, 1, 70), "all": (3, 4, 70)}[axis]
    shape = tuple(1 if n > 1 else m for n, m in zip(full, (3, 4, 70)))
    g = torch.Generator().manual_seed(12)
    base = [torch.randn(*shape, 64, generator=g).bfloat16().to(gpu).requires_grad_(True) for _ in range(3)]
    dout = torch.randn(3, 70, 4, 64, generator=g).bfloat16().to(gpu)
    wide = [t.expand(3, 4, 70, 64) for t in base]
    got = torch.autograd.grad(cross_attention(*wide), base, dout)
    dense = [t.detach().contiguous().requires_grad_(True) for t in wide]
    out = cross_attention(*dense)
    assert torch.equal(out, cross_attention(*wide))
    dims = tuple(i for i in range(3) if shape[i] == 1)
    n = math.prod(full)
    for a, b in zip(got, torch.autograd.grad(out, dense, dout)):
        want = b.double().sum(dims, keepdim=True)
        bound = 2.0 ** -8 * min(n, 32) * b.double().abs().sum(dims, keepdim=True)
        assert ((a.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("Nq,Nk", [(0, 5), (5, 0), (0, 0)])
def test_empty_axes(gpu, Nq, Nk):
    from openfold3_triangle_kernel_amd import cross_attention

    q = torch.full((2, 4, Nq, 64), float("nan"), device=gpu, dtype=torch.bfloat16, requires_grad=True)
    k = torch.ones(2, 2, Nk, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    out = cross_attention(q, k, k)
    assert out.shape == (2, Nq, 4, 64) and not out.any()
    out.sum().backward()
    assert not q.grad.any() and not k.grad.any()


def test_long_cache_offsets(gpu):
    """A cache whose byte offsets pass 32 bits: sequence-major states 2^21 apart."""
    from openfold3_triangle_kernel_amd import cross_attention

    Nk, stride = 1500, 1 << 21  # 6.3 GB
    base = torch.zeros(Nk * stride, device=gpu, dtype=torch.bfloat16)
    k = base.as_strided((1, 1, Nk, 64), (8, 8, stride, 1), 0)
    v = base.as_strided((1, 1, Nk, 64), (8, 8, stride, 1), 128)
    g = torch.Generator().manual_seed(0)
    k.copy_(torch.randn(1, 1, Nk, 64, generator=g).bfloat16())
    v.copy_(torch.randn(1, 1, Nk, 64, generator=g).bfloat16())
    for Nq in (1, 100):
        q = torch.randn(1, 1, Nq, 64, generator=g).bfloat16().to(gpu)
        with torch.no_grad():
            assert torch.equal(cross_attention(q, k, v), cross_attention(q, k.contiguous(),
                                                                         v.contiguous()))


def test_another_stream_and_graph(gpu):
    """Forward and backward on a side stream, and captured and replayed."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 2, 8, 2, 100, 700, 64, seed=11)
    mask = _mask(gpu, "tail", 2, 700, 11)
    dout = torch.randn(2, 100, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)

    def step(ops):
        leaves = [t.detach().requires_grad_(True) for t in ops]
        out = cross_attention(*leaves, mask)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = step((q, k, v))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step((q, k, v))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ops = [t.clone() for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step(ops)
    for seed in range(4):
        new = _make(gpu, 2, 8, 2, 100, 700, 64, seed=20 + seed)
        for t, n in zip(ops, new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step(new)):
            assert torch.equal(a, b)


def test_refusals(gpu):
    from openfold3_triangle_kernel_amd import cross_attention

    def ops(B=1, H=2, Hk=2, Nq=4, Nk=8, D=64, dtype=torch.bfloat16):
        return [torch.zeros(B, h, n, D, device=gpu, dtype=dtype) for h, n in ((H, Nq), (Hk, Nk), (Hk, Nk))]

    for args, match in (
            ((*ops(dtype=torch.float32), None), "BF16 or FP16"),
            ((*ops(D=136), None), "D<=128"),
            ((*ops(H=3), None), "multiple"),
            ((ops()[0], ops()[1], ops(Nk=9)[2], None), "one shape"),
            ((ops(B=2)[0], *ops()[1:], None), "batch prefix"),
            ((*ops(), torch.zeros(7, device=gpu)), "broadcast"),
            ((*ops(), torch.zeros(8, device=gpu, dtype=torch.int32)), "boolean"),
            ((*ops(), torch.zeros(8)), "one device"),
            ((*ops(), torch.zeros(8, device=gpu, requires_grad=True)), "must not require"),
            ((*ops(), None, 0.0), "scale"),
            ((*ops(), None, float("inf")), "scale"),
            ((*ops(), None, 1e-31), "scale"),
            ((*ops(), None, torch.ones((), device=gpu)), "scale")):
        with pytest.raises(ValueError, match=match):
            cross_attention(*args)
    half = [t.requires_grad_(True) for t in ops(dtype=torch.float16)]
    with pytest.raises(ValueError, match="gradients need BF16"):
        cross_attention(*half)
    with torch.no_grad():
        cross_attention(*half)


def test_prefixes_and_shared_operands(gpu):
    """No batch axis, more than one, and one tensor in several places."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 6, 4, 2, 33, 70, 64, seed=13)
    mask = _mask(gpu, "random", 6, 70, 13)
    with torch.no_grad():
        want = cross_attention(q, k, v, mask)
        one = cross_attention(q[2], k[2], v[2], mask[2])
        many = cross_attention(*(t.view(1, 2, 3, *t.shape[1:]) for t in (q, k, v)), mask.view(1, 2, 3, 70))
    assert one.shape == (33, 4, 64) and torch.equal(one, want[2])
    assert many.shape == (1, 2, 3, 33, 4, 64) and torch.equal(many.view_as(want), want)
    dout = torch.randn(6, 33, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu)
    s, qs = k.clone().requires_grad_(True), q.clone().requires_grad_(True)
    gq, gs = torch.autograd.grad(cross_attention(qs, s, s, mask), (qs, s), dout)
    parts = [t.clone().requires_grad_(True) for t in (q, k, k)]
    dq, dk, dv = torch.autograd.grad(cross_attention(*parts, mask), parts, dout)
    assert torch.equal(gq, dq) and torch.equal(gs, dk + dv)


def test_two_calls_at_once(gpu):
    """Calls that overlap on two streams, each with its own workspace."""
    from openfold3_triangle_kernel_amd import cross_attention

    cases = [_make(gpu, 2, 16, 4, 200, 3000, 64, seed=s) for s in (1, 2)]
    dout = torch.randn(2, 200, 16, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)

    def step(ops):
        leaves = [t.detach().requires_grad_(True) for t in ops]
        out = cross_attention(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(cases[i]))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


COMMON = [
    # B, H, Hk, Nq, Nk, D, mask, what K and V have in common (of the operands' deviation)
    (1, 2, 1, 30, 700, 64, "none", 0.0), (1, 2, 1, 30, 700, 64, "none", 1.0),
    (2, 4, 1, 16, 1500, 128, "tail", 1.0),  # few rows, splits joined in memory
    (1, 1, 1, 40, 3000, 64, "add", 5.0),
    (2, 4, 2, 200, 333, 128, "tail", 1.0), (2, 4, 2, 200, 333, 80, "add", 5.0),  # two wave groups
    (1, 1, 1, 300, 2000, 96, "none", 5.0), (1, 1, 1, 140, 9000, 32, "random", 2.0),  # splits
    (2, 64, 64, 520, 65, 64, "none", 2.0),  # 256 rows a workgroup
    (2, 40, 40, 260, 190, 128, "tail", 2.0),
]


def _heads_in_common(dev, B, H, Hk, Nq, Nk, D, off, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, H, Nq, D, generator=g)
    k, v = (torch.randn(B, Hk, Nk, D, generator=g) + off * torch.randn(1, Hk, 1, D, generator=g)
            for _ in range(2))
    return [t.bfloat16().to(dev) for t in (q, k, v)]


def _rounding_variances(q, k, v, mask, scale, do):
    """Outputs and gradients in 64 bits, and the squared errors to expect of them when
    P, dS and every result are rounded to BF16, each rounding an error of its own of
    mean square u^2 / 3 (uniform at the largest step of a value).  The output is a mean
    of V with weights that sum to 1, so an error d_j of p_j gives p_j d_j (v_j - o) in the
    output and p_j d_j (dP_j - delta) = d_j dS_j in delta; no rounding of the output
    enters delta."""
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1:3]
    u3 = (2.0 ** -8) ** 2 / 3
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    do = do.transpose(1, 2)
    ke, ve = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    s = scale * q @ ke.transpose(-1, -2)
    if mask is not None:
        m = mask.cpu().expand(B, Nk)[:, None, None]
        s = s.masked_fill(~m, float("-inf")) if m.dtype == torch.bool else s + m.double()
    p = torch.softmax(s, -1)
    o = p @ ve
    ds = p * (do @ ve.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    group = lambda t: t.reshape(B, Hk, H // Hk, Nk, D).sum(2)  # noqa: E731
    dq, dk = scale * ds @ ke, group(scale * ds.transpose(-1, -2) @ q)
    dv = group(p.transpose(-1, -2) @ do)
    p2, ds2 = p.square(), ds.square()
    delta = ds2.sum(-1, keepdim=True)  # of u^2 / 3
    # sum_j p_j^2 (v_j - o)^2
    spread = p2 @ ve.square() - 2 * o * (p2 @ ve) + o.square() * p2.sum(-1, keepdim=True)
    eo = o.square() + spread.clamp_min(0)
    edq = dq.square() + scale ** 2 * (ds2 @ ke.square() + delta * (p @ ke).square())
    edk = dk.square() + group(scale ** 2 * (ds2 + delta * p2).transpose(-1, -2) @ q.square())
    edv = dv.square() + group(p2.transpose(-1, -2) @ do.square())
    return ([o.transpose(1, 2), dq, dk, dv], [u3 * t.sum().item() for t in (eo, edq, edk, edv)])


@pytest.mark.parametrize("host", [True, False], ids=["cpp", "python"])
@pytest.mark.parametrize("case", COMMON, ids=str)
def test_gradients_beside_common_components(gpu, monkeypatch, case, host):
    """What keys and values have in common cancels between dO V^T and delta, and leaves
    no rounding of the output in the gradients.  Root mean squares over all elements
    against those expected; a quarter more for the sample's scatter and the 32-bit sums
    (the expected ones are 1.2 to 1.4 times too high already: a value's last place is
    smaller against it than u, but for powers of two)."""
    from openfold3_triangle_kernel_amd import _native, cross_attention

    if not host:
        monkeypatch.setattr(_native, "_HOST", False)
    B, H, Hk, Nq, Nk, D, mk, off = case
    q, k, v = (t.requires_grad_(True) for t in _heads_in_common(gpu, B, H, Hk, Nq, Nk, D, off, 31))
    mask = _mask(gpu, mk, B, Nk, 31)
    do = torch.randn(B, Nq, H, D, generator=torch.Generator().manual_seed(32)).bfloat16().to(gpu)
    want, expected = _rounding_variances(q, k, v, mask, 1 / math.sqrt(D), do)
    out = cross_attention(q, k, v, mask)
    got = [out.detach(), *torch.autograd.grad(out, (q, k, v), do)]
    for g, w, e, name in zip(got, want, expected, ("out", "dq", "dk", "dv")):
        err = (g.double().cpu() - w).square().sum().item()
        assert err <= 1.25 ** 2 * e, f"{name}: {(err / e) ** 0.5:.2f} of the expected error"


def test_shadow_policy(gpu, monkeypatch):
    """Without the residual (TURBOPAIRFORMER_SR_SHADOW=0) the same output and dV, delta
    from the rounded output, on both host paths; another value is refused."""
    from openfold3_triangle_kernel_amd import _native, cross_attention

    q, k, v = (t.requires_grad_(True) for t in _heads_in_common(gpu, 1, 2, 1, 130, 200, 64, 2.0, 33))
    do = torch.randn(1, 130, 2, 64, generator=torch.Generator().manual_seed(34)).bfloat16().to(gpu)

    def run():
        out = cross_attention(q, k, v)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), do)]

    want, tol = _reference(q, k, v, None, 1 / 8.0, do)  # its delta counts the output's rounding
    runs = {}
    for shadow in ("1", "0"):
        monkeypatch.setenv("TURBOPAIRFORMER_SR_SHADOW", shadow)
        for host in (None, False):
            with monkeypatch.context() as m:
                if host is False:
                    m.setattr(_native, "_HOST", False)
                runs[shadow, host] = run()
        assert all(torch.equal(a, b) for a, b in zip(runs[shadow, None], runs[shadow, False]))
    with_, without = runs["1", None], runs["0", None]
    _check(without, want, tol)
    assert torch.equal(with_[0], without[0]) and torch.equal(with_[3], without[3])
    assert not torch.equal(with_[1], without[1])
    monkeypatch.setenv("TURBOPAIRFORMER_SR_SHADOW", "2")
    with pytest.raises(ValueError, match="must be 0 or 1"):
        cross_attention(q, k, v)
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v), with_[0])


@pytest.mark.parametrize("Nq", [1, 100])
def test_masks_in_64_bits(gpu, Nq):
    """Finite values past the 32-bit range are finite still: at the lowest a state is not
    dropped, at the highest it does not make its rows NaN."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 2, 2, 2, Nq, 130, 64, seed=8)
    ends = torch.finfo(torch.float64).min, torch.finfo(torch.float64).max
    wide = torch.randn(2, 130, dtype=torch.float64, generator=torch.Generator().manual_seed(8)).to(gpu)
    wide[0, 7], wide[0, 9], wide[1] = float("-inf"), ends[0], ends[0]
    narrow = wide.clamp(torch.finfo(torch.float32).min, torch.finfo(torch.float32).max).float()
    narrow[0, 7] = float("-inf")
    with torch.no_grad():
        out = cross_attention(q, k, v, wide)
        assert torch.equal(out, cross_attention(q, k, v, narrow))
        assert out[1].any()  # live states, not a row of zeros
        wide[1, 5], narrow[1, 5] = ends[1], torch.finfo(torch.float32).max
        out = cross_attention(q, k, v, wide)
        assert torch.equal(out, cross_attention(q, k, v, narrow)) and torch.isfinite(out).all()
        wide[1, 6] = float("nan")
        assert cross_attention(q, k, v, wide)[1].isnan().all()


@pytest.mark.parametrize("host", [True, False], ids=["cpp", "python"])
def test_more_rows_than_a_launch_holds_are_refused(gpu, monkeypatch, host):
    from openfold3_triangle_kernel_amd import _native, cross_attention

    if not host:
        monkeypatch.setattr(_native, "_HOST", False)
    one = torch.zeros(1, 1, 1, 8, device=gpu, dtype=torch.bfloat16)
    wide = one.expand(1 << 24, -1, -1, -1)
    with pytest.raises(ValueError, match="too many"):
        cross_attention(wide, wide, wide)
    states = one.expand(1 << 11, -1, 1 << 20, -1)  # the dK / dV launch
    with pytest.raises(ValueError, match="too many states"):
        cross_attention(one.expand(1 << 11, -1, -1, -1).clone().requires_grad_(True), states, states)


@pytest.mark.parametrize("mk", ["none", "random", "add"])
@pytest.mark.parametrize("scale", [0.02, 1, 4.0])
@pytest.mark.parametrize("B,H,Hk,Nq,Nk,D", [(2, 4, 2, 3, 400, 64), (2, 2, 1, 130, 150, 40)])
def test_explicit_scales(gpu, B, H, Hk, Nq, Nk, D, scale, mk):
    """Scales other than the default in both directions, whole numbers too; additive
    values are added after the scale."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = (t.requires_grad_(True)
               for t in _make(gpu, B, H, Hk, Nq, Nk, D, seed=14, qscale=0.5))
    mask = _mask(gpu, mk, B, Nk, 14)
    dout = torch.randn(B, Nq, H, D, generator=torch.Generator().manual_seed(15)).bfloat16().to(gpu)
    want, tol = _reference(q, k, v, mask, scale, dout)
    out = cross_attention(q, k, v, mask, scale)
    _check([out, *torch.autograd.grad(out, (q, k, v), dout)], want, tol)


@pytest.mark.parametrize("scale", [1e-29, 1e-10, 1e6, 1e29])
def test_scales_of_the_whole_range(gpu, scale):
    """q carries the scale's inverse: the products are those of the default scale."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 1, 2, 1, 70, 90, 64, seed=16)
    mask = _mask(gpu, "add", 1, 90, 16)
    power = round(math.log2(0.125 / scale))
    qs = (q.float() * 2.0 ** power).bfloat16().requires_grad_(True)
    k, v = k.requires_grad_(True), v.requires_grad_(True)
    dout = torch.randn(1, 70, 2, 64, generator=torch.Generator().manual_seed(17)).bfloat16().to(gpu)
    want, tol = _reference(qs, k, v, mask, scale, dout)
    out = cross_attention(qs, k, v, mask, scale)
    _check([out, *torch.autograd.grad(out, (qs, k, v), dout)], want, tol)


@pytest.mark.parametrize("scale", [0.125, 4.0])
@pytest.mark.parametrize("Nq,Nk", [(1, 90), (5, 1500), (1, 6000), (130, 200), (200, 3000)])
def test_scores_of_minus_infinity(gpu, Nq, Nk, scale):
    """A live state whose score is -inf has no weight; a row that has only such is NaN, as
    0 / 0 is, and no row without a state (which is 0)."""
    from openfold3_triangle_kernel_amd import cross_attention

    q, k, v = _make(gpu, 2, 4, 2, Nq, Nk, 64, seed=18)
    q[..., 0], k[..., 0] = q[..., 0].abs() + 0.5, -k[..., 0].abs() - 0.5
    whole = _mask(gpu, "random", 2, Nk, 18)
    whole[:, 0] = True
    add = torch.where(whole, 0.25, float("-inf"))
    with torch.no_grad():
        # The first states (whole tiles of them among many), and some of the others.
        far = torch.zeros(2, 2, Nk, dtype=torch.bool, device=gpu)
        far[:, :, :Nk // 3] = True
        far[:, :, -1] = True
        ks = k.clone()
        ks[..., 0] = torch.where(far, float("-inf"), ks[..., 0])
        for mask in (None, whole, add):
            kept = torch.ones(2, Nk, dtype=torch.bool, device=gpu) if mask is None else whole
            want, tol = _reference(q, k, v, kept & ~far[:, 0], scale)
            _check([cross_attention(q, ks, v, mask, scale)], want, tol)
        for mask in (None, whole, add):
            qi = q.clone()
            qi[1, 2, Nq // 2, 0] = float("inf")
            out, clean = cross_attention(qi, k, v, mask, scale), cross_attention(q, k, v, mask, scale)
            hit = torch.zeros(2, Nq, 4, dtype=torch.bool, device=gpu)
            hit[1, Nq // 2, 2] = True
            assert out[hit].isnan().all() and torch.equal(out[~hit], clean[~hit])
        none = whole.clone()
        none[1] = False
        assert not cross_attention(qi, k, v, none, scale)[1].any()


@pytest.mark.parametrize("host", [True, False], ids=["cpp", "python"])
def test_sequences_far_apart(gpu, monkeypatch, host):
    """Caches whose sequences or heads lie 2^24 elements apart are read in place, and by the
    C++ host path where it is there."""
    import sys

    from openfold3_triangle_kernel_amd import _native, cross_attention

    module = sys.modules["openfold3_triangle_kernel_amd.cross_attention"]
    q, k, v = _make(gpu, 2, 4, 2, 3, 200, 64, seed=19)
    far = torch.zeros(2, 1 << 24, device=gpu, dtype=torch.bfloat16)
    kc, vc = (far[:, at:at + 2 * 200 * 64].view(2, 2, 200, 64) for at in (0, 1 << 16))
    kc.copy_(k), vc.copy_(v)
    with torch.no_grad():
        want = cross_attention(q, k, v)
        if host:
            monkeypatch.setattr(module, "_check", lambda *args: pytest.fail("not the C++ host path"))
        else:
            monkeypatch.setattr(_native, "_HOST", False)
        assert torch.equal(cross_attention(q, kc, vc), want)
        heads = [t.transpose(0, 1) for t in (kc, vc)]
        assert torch.equal(cross_attention(q[:, :2], *heads),
                           cross_attention(q[:, :2], *(t.contiguous() for t in heads)))

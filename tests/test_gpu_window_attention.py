"""Causal self-attention with a window and sinks against the formulas in 64 bits.

Tolerances count roundings.  With u = finfo(type).eps / 2: the probabilities enter the
second product rounded (u each), outputs are rounded once (u), and the scores carry D + 4
roundings of 32 bits, ds = (D + 4) 2^-24 scale sum |q||k|, which a softmax turns into a
relative error of at most 2 ds (numerator and sum); the exponential and the sums add 2^-20
and (N / 32 + 64) 2^-24.  FP16 probabilities below 2^-14 are subnormal: 2^-25 each, the
largest being at least 1.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

_T = {"bf16": torch.bfloat16, "fp16": torch.float16}


def seen(rows, states, window, sinks):
    """[len(rows), states]: what tokens at the positions ``rows`` see."""
    col, row = torch.arange(states), rows[:, None]
    see = col <= row
    if window:
        see = see & ((row - col < window) | (col < sinks))
    return see


def reference(q, k, v, see, scale, dout=None):
    """(out, dq, dk, dv) and their bounds of q [H, R, D] on k, v [Hk, S, D] in 64 bits;
    see [R, S]."""
    u = torch.finfo(q.dtype).eps / 2
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    (H, R, D), (Hk, S) = q.shape, k.shape[:2]
    G = H // Hk
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    ke, ve = (t.repeat_interleave(G, 0) for t in (k, v))
    s = (scale * q @ ke.transpose(-1, -2)).masked_fill(~see, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ ve
    ds_ = (D + 4) * 2.0 ** -24 * (scale * (q.abs() @ ke.abs().transpose(-1, -2))).amax(-1, keepdim=True)
    rel = 2 * ds_ + 2.0 ** -20 + (S / 32 + 64) * 2.0 ** -24
    few = see.sum(-1)[:, None]
    eo = u * o.abs() + (u + rel) * (p @ ve.abs()) * (1 + u) + (few > 0) * sub * (
        see.double() @ ve.abs() + 2)
    outs, errs = [o], [eo]
    if dout is None:
        return outs, errs
    do = dout.detach().double().cpu()
    dp = do @ ve.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    edelta = (do.abs() * eo).sum(-1, keepdim=True) + D * 2.0 ** -24 * (do.abs() * o.abs()).sum(-1, keepdim=True)
    edp = (D + 4) * 2.0 ** -24 * (do.abs() @ ve.abs().transpose(-1, -2))
    ds = p * (dp - delta)
    eds = (u + rel) * ds.abs() * (1 + u) + p * (edelta + edp) * (1 + u + rel)
    sums = (G * R / 16 + S / 16 + 64) * 2.0 ** -24
    group = lambda t: t.reshape(Hk, G, S, D).sum(1)  # noqa: E731
    dq, dk = scale * ds @ ke, group(scale * ds.transpose(-1, -2) @ q)
    dv = group(p.transpose(-1, -2) @ do)
    edq = u * dq.abs() + scale * ((eds + sums * ds.abs()) @ ke.abs()) * (1 + u)
    edk = u * dk.abs() + group(scale * (eds + sums * ds.abs()).transpose(-1, -2) @ q.abs()) * (1 + u)
    edv = u * dv.abs() + group(((u + rel + sums) * p).transpose(-1, -2) @ do.abs()) * (1 + u)
    return outs + [dq, dk, dv], errs + [edq, edk, edv]


def check(got, want, tol, names=("out", "dq", "dk", "dv")):
    for g, w, t, name in zip(got, want, tol, names):
        g = g.detach().double().cpu()
        assert g.shape == w.shape, name
        over = ((g - w).abs() - t - 1e-30).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"


def make(dev, B, H, Hk, N, D, dtype=torch.bfloat16, layout="head", seed=0, qscale=1.5):
    g = torch.Generator().manual_seed(seed)

    def heads(h, scale=1.0):
        if layout == "seq":
            return torch.randn(B, N, h, D, generator=g).mul(scale).to(dtype).to(dev).transpose(1, 2)
        if layout == "fused":  # a slice of a wider projection
            t = torch.randn(B, N, h, 2 * D, generator=g).mul(scale).to(dtype).to(dev)
            return t[..., D:].transpose(1, 2)
        return torch.randn(B, h, N, D, generator=g).mul(scale).to(dtype).to(dev)

    return heads(H, qscale), heads(Hk), heads(Hk)


def _mask(dev, kind, B, N, seed=0):
    g = torch.Generator().manual_seed(100 + seed)
    if kind == "none":
        return None
    if kind == "tail":
        return (torch.arange(N) < N - torch.randint(0, N // 2 + 1, (B, 1), generator=g)).to(dev)
    m = torch.rand(B, N, generator=g) < (0.4 if kind == "random" else 0.7)
    if kind == "empty":
        m[0] = False
    if kind == "head":  # the first rows see nothing
        m[:, :N // 2] = False
    return m.to(dev)


def _all(q, k, v, mask, window, sinks, dout=None):
    B, H, N, D = q.shape
    see = seen(torch.arange(N), N, window, sinks)
    parts = []
    for b in range(B):
        s = see if mask is None else see & mask.expand(B, N)[b].cpu()
        parts.append(reference(q[b], k[b], v[b], s, 1 / math.sqrt(D),
                               None if dout is None else dout[b].transpose(0, 1)))
    outs, errs = ([torch.stack(x) for x in zip(*(p[i] for p in parts))] for i in (0, 1))
    outs[0], errs[0] = outs[0].transpose(1, 2), errs[0].transpose(1, 2)
    return outs, errs


FORWARD = [
    # B, H, Hk, N, D, window, sinks, type, layout, mask
    (1, 1, 1, 1, 8, 0, 0, "bf16", "head", "none"),
    (1, 1, 1, 2, 20, 1, 0, "fp16", "head", "none"),
    (2, 8, 8, 77, 64, 0, 0, "fp16", "seq", "none"),
    (3, 8, 2, 33, 128, 5, 3, "bf16", "seq", "tail"),
    (2, 4, 2, 130, 40, 64, 0, "bf16", "fused", "random"),
    (2, 6, 2, 200, 96, 63, 70, "fp16", "head", "head"),
    (1, 3, 1, 300, 80, 65, 1, "bf16", "seq", "empty"),
    (2, 4, 4, 513, 128, 0, 0, "bf16", "head", "tail"),
    (1, 7, 1, 400, 72, 100, 64, "bf16", "head", "none"),
    (1, 2, 2, 1500, 64, 300, 7, "bf16", "seq", "random"),  # parts of the states
    (1, 1, 1, 2049, 32, 0, 0, "fp16", "head", "none"),
    (1, 1, 1, 1100, 128, 1, 500, "bf16", "head", "none"),
    (1, 4, 1, 700, 48, 2000, 9, "bf16", "seq", "head"),  # a window past the tokens
    (2, 64, 64, 600, 64, 128, 4, "bf16", "head", "none"),
    (4, 64, 64, 600, 32, 128, 4, "bf16", "head", "none"),  # 256 rows a workgroup
    (4, 64, 64, 513, 32, 0, 0, "fp16", "seq", "random"),
    (1, 40, 1, 70, 64, 9, 2, "bf16", "seq", "none"),
    (1, 300, 1, 20, 32, 4, 1, "fp16", "head", "tail"),
    (3, 1, 1, 1, 128, 1, 0, "bf16", "seq", "tail"),
]


@pytest.mark.parametrize("case", FORWARD, ids=str)
def test_forward(gpu, case):
    from openfold3_triangle_kernel_amd import window_attention

    B, H, Hk, N, D, window, sinks, t, layout, mk = case
    q, k, v = make(gpu, B, H, Hk, N, D, _T[t], layout)
    mask = _mask(gpu, mk, B, N)
    with torch.no_grad():
        out = window_attention(q, k, v, window or None, sinks, mask)
    assert out.shape == (B, N, H, D) and out.is_contiguous()
    check([out], *_all(q, k, v, mask, window, sinks))
    if mk == "empty":
        assert not out[0].any()
    if mk == "head":
        assert not out[:, :N // 2].any()


BACKWARD = [
    # B, H, Hk, N, D, window, sinks, layout, mask
    (1, 1, 1, 1, 8, 0, 0, "head", "none"),
    (2, 4, 2, 65, 64, 0, 0, "seq", "tail"),
    (2, 4, 4, 100, 32, 17, 3, "head", "random"),
    (2, 8, 2, 257, 64, 64, 0, "fused", "empty"),
    (3, 3, 1, 190, 80, 50, 40, "seq", "head"),
    (1, 2, 2, 130, 96, 1, 0, "head", "none"),
    (2, 4, 2, 333, 128, 100, 5, "seq", "tail"),
    (1, 7, 1, 300, 128, 0, 0, "head", "none"),
    (1, 6, 1, 700, 40, 30, 200, "head", "random"),  # two tiles of sinks, in parts
    (1, 1, 1, 1500, 64, 129, 1, "seq", "none"),
    (1, 2, 1, 1300, 128, 64, 130, "seq", "none"),
    (1, 5, 1, 400, 20, 3, 1, "head", "none"),
    (1, 40, 1, 40, 32, 9, 2, "seq", "none"),
    (1, 2, 2, 260, 72, 500, 9, "head", "tail"),
    (8, 64, 64, 130, 24, 50, 2, "head", "tail"),  # 256 rows a workgroup
    (1, 2, 1, 900, 64, 5, 600, "head", "none"),  # most tokens are sinks
    (1, 2, 1, 300, 32, 5, 300, "seq", "tail"),  # all are
    (2, 200, 1, 20, 64, 4, 1, "head", "none"),  # more heads to a kv head than a tile has rows
]


@pytest.mark.parametrize("case", BACKWARD, ids=str)
def test_backward(gpu, case):
    from openfold3_triangle_kernel_amd import window_attention

    B, H, Hk, N, D, window, sinks, layout, mk = case
    q, k, v = (t.requires_grad_(True) for t in make(gpu, B, H, Hk, N, D, layout=layout, seed=3))
    mask = _mask(gpu, mk, B, N, 3)
    dout = torch.randn(B, N, H, D, generator=torch.Generator().manual_seed(9)).bfloat16().to(gpu)
    want, tol = _all(q, k, v, mask, window, sinks, dout)
    run = lambda: window_attention(q, k, v, window or None, sinks, mask)  # noqa: E731
    out = run()
    grads = torch.autograd.grad(out, (q, k, v), dout)
    check([out, *grads], want, tol)
    for a, b in zip(grads, torch.autograd.grad(run(), (q, k, v), dout)):
        assert torch.equal(a, b)
    if mask is not None:
        dead = ~mask[:, None, :, None]
        assert not (grads[1] * dead).any() and not (grads[2] * dead).any()


@pytest.mark.parametrize("case", [
    # Parts of the states' rows that take turns: the last one shorter than the others.
    (10, 16, 8, 640, 32, 400, 3, "seq", "none"),
    (20, 9, 3, 600, 64, 400, 130, "head", "tail"),
    (5, 16, 4, 2000, 128, 470, 1, "seq", "none"),
], ids=str)
def test_backward_in_uneven_parts(gpu, case):
    test_backward(gpu, case)


def test_gradients_against_differences(gpu):
    """Directional differences of the 64-bit formula at the BF16 operands: the gradient's own
    roundings (2^-9 relative, a few of them) bound the deviation."""
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = (t.requires_grad_(True) for t in make(gpu, 1, 2, 1, 50, 64, seed=5))
    mask = _mask(gpu, "tail", 1, 50, 5)
    dout = torch.randn(1, 50, 2, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    grads = torch.autograd.grad(window_attention(q, k, v, 20, 2, mask), (q, k, v), dout)
    base = [t.detach().double().cpu() for t in (q, k, v)]

    def loss(ops):
        return (_all(*ops, mask, 20, 2)[0][0] * dout.double().cpu()).sum().item()

    for n in range(3):
        g = grads[n].double().cpu()
        step = g / g.norm()
        ops = [list(base), list(base)]
        ops[0][n], ops[1][n] = base[n] + 1e-5 * step, base[n] - 1e-5 * step
        slope = (loss(ops[0]) - loss(ops[1])) / 2e-5
        assert abs(slope - g.norm().item()) <= 2.0 ** -7 * g.norm().item()


def test_shared_heads_and_common_parts(gpu):
    """Values with much in common pass exactly but for the outputs' rounding."""
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = make(gpu, 1, 4, 2, 300, 64, seed=2)
    v = torch.full_like(v, 3.0)
    out = window_attention(q, k, v, 40, 3)
    assert torch.equal(out, torch.full_like(out, 3.0))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("N,D,window,sinks", [(70, 64, None, 0), (200, 128, 50, 3), (150, 96, 20, 0),
                                              (130, 32, 7, 100), (600, 64, 128, 4), (260, 32, 128, 4)])
def test_what_a_row_does_not_see_never_reaches_it(gpu, bad, N, D, window, sinks):
    """Whatever a token holds, the rows that do not see it, and the gradients of the states
    that its row does not see, are those of zeros there; dropped tokens reach nothing."""
    from openfold3_triangle_kernel_amd import window_attention

    heads = {600: (64, 64), 260: (256, 128)}.get(N, (4, 2))  # (260: 256 rows a workgroup)
    q, k, v = make(gpu, 2, *heads, N, D, seed=7)
    at = N // 2
    see = seen(torch.arange(N), N, window or 0, sinks).to(gpu)
    dout = torch.randn(2, N, heads[0], D, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)

    def run(q, k, v, mask=None, dout=dout):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = window_attention(*leaves, window, sinks, mask)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    for what in range(3):
        ops, clean = [t.clone() for t in (q, k, v)], [t.clone() for t in (q, k, v)]
        ops[what][1, 1, at, 3] = bad
        clean[what][1, 1, at, 3] = 0.0
        got, want = run(*ops), run(*clean)
        out, dq, dk, dv = [torch.equal(a[0], b[0]) for a, b in zip(got, want)]
        assert out and dq and dk and dv  # the other batch entry
        if what:  # rows before the token, or past its window
            blind = ~see[:, at]
            assert torch.equal(got[0][1, blind], want[0][1, blind])
            assert torch.equal(got[1][1][:, blind], want[1][1][:, blind])
            assert torch.isfinite(got[0][1, blind]).all()
            mine = got[0][1][see[:, at]]
            assert not torch.isfinite(mine).all()
            if what == 2:  # every row that sees it, in the heads of its kv head
                g = heads[0] // heads[1]
                hit = mine[:, g:2 * g, 3]
                assert (hit.isnan() if bad != bad else hit == bad).all()
                mine[:, g:2 * g, 3] = 0
                assert torch.isfinite(mine).all()
        else:  # one row: itself, and the gradients of the states that it sees
            rows = torch.ones(N, dtype=torch.bool, device=gpu)
            rows[at] = False
            assert torch.equal(got[0][1, rows], want[0][1, rows])
            assert torch.equal(got[1][1][:, rows], want[1][1][:, rows])
            for i in (2, 3):
                assert torch.equal(got[i][1][:, ~see[at]], want[i][1][:, ~see[at]])
    # An upstream gradient's row.
    hurt, none = dout.clone(), dout.clone()
    hurt[1, at, 1, 3], none[1, at, 1, 3] = bad, 0.0
    got, want = run(q, k, v, dout=hurt), run(q, k, v, dout=none)
    for i in (2, 3):
        assert torch.equal(got[i][1][:, ~see[at]], want[i][1][:, ~see[at]])
    # A dropped token's key and value.
    mask = torch.ones(2, N, dtype=torch.bool, device=gpu)
    mask[1, at] = False
    runs = []
    for fill in (0.0, bad):
        ks, vs = k.clone(), v.clone()
        ks[1, :, at], vs[1, :, at] = fill, fill
        runs.append(run(q, ks, vs, mask))
    for a, b in zip(*runs):
        assert torch.isfinite(b).all() and torch.equal(a, b)


@pytest.mark.parametrize("N,window,at", [(40, None, 10), (40, 8, 10), (64, None, 0), (1500, 1, 700), (1500, 5, 1499),
                                         (1500, None, 3)])
def test_a_score_that_is_nan_reaches_every_value_gradient(gpu, N, window, at):
    """Rows that see a NaN key have NaN probabilities: so have the value gradients of all
    states that such a row sees, whether the row's states lie in one tile or in many."""
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = make(gpu, 1, 4, 2, N, 32, seed=9)
    k[0, 0, at, 5] = float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    dout = torch.randn(1, N, 4, 32, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    out = window_attention(*leaves, window)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    see = seen(torch.arange(N), N, window, 0).to(gpu)
    rows = see[:, at]                   # that see the key
    states = see[rows].any(0)           # that one of these sees
    assert out[0, rows, :2].isnan().all() and torch.isfinite(out[0, ~rows]).all()
    assert dq[0, :2, rows].isnan().all() and torch.isfinite(dq[0, :2, ~rows]).all()
    for t in (dk, dv):
        assert t[0, 0, states].isnan().all()
        assert torch.isfinite(t[0, 0, ~states]).all()
    for t in (out[0, :, 2:], dq[0, 2:], dk[0, 1], dv[0, 1]):
        assert torch.isfinite(t).all()


def test_rows_whose_scores_are_all_minus_infinity(gpu):
    """They are NaN, unlike rows that see no state."""
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = make(gpu, 1, 2, 1, 100, 64, seed=3)
    q[0, 1, 40] = -1.0
    k[0, 0, :41] = 1.0
    k[0, 0, :41, 0] = float("inf")
    q[0, 0, 40] = 0.0  # 0 times infinity: NaN as well
    mask = torch.ones(1, 100, dtype=torch.bool, device=gpu)
    mask[0, :10] = False
    out = window_attention(q, k, v, None, 0, mask)
    assert out[0, 40].isnan().all() and not out[0, :10].any()
    assert torch.isfinite(out[0, :10]).all()


def test_masks_and_prefixes(gpu):
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = make(gpu, 6, 2, 1, 90, 32, seed=4)
    q, k, v = (t.reshape(2, 3, *t.shape[1:]) for t in (q, k, v))
    for m in (_mask(gpu, "random", 1, 90)[0], _mask(gpu, "random", 3, 90), _mask(gpu, "random", 2, 90)[:, None],
              _mask(gpu, "random", 90, 3).t()):
        full = m.expand(2, 3, 90).contiguous()
        want = window_attention(q, k, v, 30, 2, full)
        assert torch.equal(window_attention(q, k, v, 30, 2, m), want)
        one = window_attention(q[1, 2], k[1, 2], v[1, 2], 30, 2, full[1, 2])
        assert torch.equal(one, want[1, 2])


def test_broadcast_and_offset_operands(gpu):
    """Expanded operands sum their gradients, storage off the 16 bytes is copied."""
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = make(gpu, 1, 4, 2, 70, 64, seed=6)
    dout = torch.randn(3, 70, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    leaf = k.clone().requires_grad_(True)
    q3, v3 = q.repeat(3, 1, 1, 1), v.repeat(3, 1, 1, 1)
    out = window_attention(q3, leaf.expand(3, -1, -1, -1), v3, 20, 3)
    got, = torch.autograd.grad(out, leaf, dout)
    k3 = k.repeat(3, 1, 1, 1).requires_grad_(True)
    out3 = window_attention(q3, k3, v3, 20, 3)
    want, = torch.autograd.grad(out3, k3, dout)
    assert torch.equal(out, out3)
    # The three terms are added in BF16: two roundings of partial sums.
    assert ((got.double() - want.double().sum(0, keepdim=True)).abs()
            <= 2 * 2.0 ** -8 * want.double().abs().sum(0)).all()
    flat = torch.zeros(k.numel() + 8, device=gpu, dtype=k.dtype)
    wide = torch.zeros(1, 2, 70, 67, device=gpu, dtype=k.dtype)  # odd state stride
    wide[..., :64] = k
    plain = window_attention(q, k, v, 20, 3)
    for off in (1, 3, 4):
        shifted = flat[off:off + k.numel()].view(k.shape)
        shifted.copy_(k)
        assert torch.equal(window_attention(q, shifted, v, 20, 3), plain)
    assert torch.equal(window_attention(q, wide[..., :64], v, 20, 3), plain)


@pytest.mark.parametrize("shape", [(2, 4, 0, 64), (0, 4, 5, 64)])
def test_empty_axes(gpu, shape):
    from openfold3_triangle_kernel_amd import window_attention

    q = torch.ones(shape, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    out = window_attention(q, q, q, 3)
    assert out.shape == (shape[0], shape[2], shape[1], shape[3])
    out.sum().backward()
    assert q.grad.shape == shape


def test_long_operands(gpu):
    """States and rows whose byte offsets pass 32 bits."""
    from openfold3_triangle_kernel_amd import window_attention

    base = torch.zeros(1500 << 21, device=gpu, dtype=torch.bfloat16)  # 6.3 GB
    g = torch.Generator().manual_seed(0)
    q, k, v = (base.as_strided((1, 1, 1500, 64), (8, 8, 1 << 21, 1), 128 * i) for i in range(3))
    for t in (q, k, v):
        t.copy_(torch.randn(1, 1, 1500, 64, generator=g).bfloat16())
    dout = torch.randn(1, 1500, 1, 64, generator=g).bfloat16().to(gpu)
    runs = []
    for ops in ((q, k, v), [t.contiguous() for t in (q, k, v)]):
        leaves = [t.detach().requires_grad_(True) for t in ops]
        out = window_attention(*leaves, 200, 2)
        # (No gradient of the far operands' own order: it would be as long.)
        runs.append([out.detach()])
    assert torch.equal(runs[0][0], runs[1][0])
    far = q.detach().requires_grad_(True)
    near = q.contiguous().detach().requires_grad_(True)
    ks, vs = k.contiguous(), v.contiguous()
    a, = torch.autograd.grad(window_attention(far, ks, vs, 200, 2), far, dout)
    b, = torch.autograd.grad(window_attention(near, ks, vs, 200, 2), near, dout)
    assert torch.equal(a, b)


def test_another_stream_and_graph(gpu):
    from openfold3_triangle_kernel_amd import window_attention

    mask = _mask(gpu, "tail", 2, 700, 11)
    dout = torch.randn(2, 700, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)

    def step(ops):
        leaves = [t.detach().requires_grad_(True) for t in ops]
        out = window_attention(*leaves, 100, 3, mask)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    first = make(gpu, 2, 8, 2, 700, 64, seed=11)
    want = step(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(first)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ops = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step(ops)
    for seed in range(3):
        new = make(gpu, 2, 8, 2, 700, 64, seed=20 + seed)
        for t, n in zip(ops, new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step(new)):
            assert torch.equal(a, b)


def test_two_calls_at_once(gpu):
    """Calls that overlap on two streams, each with its own workspace."""
    from openfold3_triangle_kernel_amd import window_attention

    cases = [make(gpu, 1, 2, 2, 3000, 64, seed=s) for s in (1, 2)]
    dout = torch.randn(1, 3000, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)

    def step(ops):
        leaves = [t.detach().requires_grad_(True) for t in ops]
        out = window_attention(*leaves, 300, 4)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(cases[i]))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_half_precision_has_no_gradients(gpu):
    from openfold3_triangle_kernel_amd import window_attention

    q = torch.zeros(1, 2, 4, 64, device=gpu, dtype=torch.float16, requires_grad=True)
    with pytest.raises(ValueError, match="gradients need BF16"):
        window_attention(q, q, q)
    with torch.no_grad():
        window_attention(q, q, q)


def test_residual_policy(gpu, monkeypatch):
    """With and without what the output's rounding drops: outputs alike, gradients within
    the outputs' rounding (2^-9 of delta's terms)."""
    from openfold3_triangle_kernel_amd import window_attention

    q, k, v = (t.requires_grad_(True) for t in make(gpu, 1, 4, 2, 300, 64, seed=15))
    dout = torch.randn(1, 300, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16().to(gpu)
    runs = []
    for flag in "10":
        monkeypatch.setenv("TURBOPAIRFORMER_SR_SHADOW", flag)
        out = window_attention(q, k, v, 90, 2)
        runs.append([out, *torch.autograd.grad(out, (q, k, v), dout)])
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][3], runs[1][3])
    for a, b in zip(runs[0][1:3], runs[1][1:3]):
        assert (a - b).norm() <= 2.0 ** -6 * a.norm()

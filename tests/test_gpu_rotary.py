"""Norms of queries and keys with the position rotation against the formulas in 64 bits.

Tolerances count roundings.  u = finfo(type).eps / 2 for the one rounding of a result.  In
32 bits: a mean of D squares and its inverse root are within (D / 2 + 8) 2^-24 of their
values, an angle within 2^-22 radians (2^-25 of a turn), sine and cosine within 4 x 2^-24
more, and a pair's product sum adds 3 x 2^-24 of its terms.  Sums over rows add at most
2^-24 of their terms for each of the rows.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ANGLE = 2.0 ** -22 + 7 * 2.0 ** -24


def _make(dev, B, N, H, Hk, D, dtype, layout="seq", seed=0):
    g = torch.Generator().manual_seed(seed)

    def heads(h):
        if layout == "seq":
            return torch.randn(B, N, h, D, generator=g).to(dtype).to(dev).transpose(1, 2)
        if layout == "fused":  # a slice of a wider projection, off the 16 bytes
            return torch.randn(B, N, h, 2 * D + 1, generator=g).to(dtype).to(dev)[..., D:2 * D].transpose(1, 2)
        return torch.randn(B, h, N, D, generator=g).to(dtype).to(dev)

    return heads(H), heads(Hk), g


def _frequencies(half, dev):
    return (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).to(dev)


def _turn(x, positions, freq, inter, back=False):
    """(R x, |R| |x|): the rotation in 64 bits and the size of its terms."""
    half = len(freq)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if inter else (
        slice(0, half), slice(half, 2 * half))
    t = positions.double()[:, None, :, None] * freq
    c, s = t.cos(), t.sin() * (-1 if back else 1)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def _reference(x, dy, positions, freq, w, eps, inter):
    """(y, bound) and, with dy, (dx, bound), (dw, bound) of one side."""
    u = torch.finfo(x.dtype).eps / 2
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    D = x.shape[-1]
    f = torch.zeros(0, dtype=torch.float64) if freq is None else freq.double().cpu()
    x = x.detach().double().cpu()
    positions = positions.cpu()
    wd = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
    en = (D / 2 + 8) * 2.0 ** -24 if eps is not None else 0.0
    r = torch.ones_like(x[..., :1]) if eps is None else (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * r
    z = xh * wd
    y, size = _turn(z, positions, f, inter)
    out = [(y, u * y.abs() + (1 + u) * (en * (size + z.abs()) + _ANGLE * size) + sub)]
    if dy is None:
        return out
    dz, dsize = _turn(dy.double().cpu(), positions, f, inter, back=True)
    edz = _ANGLE * dsize
    g, eg = dz * wd, (edz + 2.0 ** -24 * dz.abs()) * wd.abs()
    if eps is None:
        return out + [(g, u * g.abs() + (1 + u) * eg + sub), None]
    m = (g * xh).mean(-1, keepdim=True)
    dx = r * (g - xh * m)
    terms = g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)
    e = r * (eg + xh.abs() * (eg * xh.abs()).mean(-1, keepdim=True) + (3 * en + D * 2.0 ** -24) * terms)
    out.append((dx, u * dx.abs() + (1 + u) * e + sub))
    if w is None:
        return out + [None]
    uw = torch.finfo(w.dtype).eps / 2
    dw = (dz * xh).sum((0, 1, 2))
    rows = x.numel() // D
    ew = (edz * xh.abs() + (en + (rows + 2) * 2.0 ** -24) * (dz * xh).abs()).sum((0, 1, 2))
    return out + [(dw, uw * dw.abs() + (1 + uw) * ew + (2.0 ** -25 if w.dtype == torch.float16 else 0.0))]


def _check(got, want, name):
    want, bound = want
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    over = ((got - want).abs() - bound - 1e-30).max().item()
    assert over <= 0, f"{name}: {over:.3e} over the bound"


CASES = [
    # B, N, H, Hk, D, half, type, weights, layout, norm, interleaved, positions
    (1, 1, 1, 1, 1, 0, "fp32", "fp32", "head", True, False, "none"),
    (1, 1, 1, 1, 2, 1, "bf16", "fp32", "head", True, True, "far"),
    (2, 3, 4, 2, 7, 3, "fp32", "fp32", "fused", True, False, "far"),
    (2, 5, 3, 1, 20, 5, "bf16", "bf16", "seq", True, True, "int32"),
    (1, 77, 8, 8, 64, 32, "fp16", "fp32", "seq", True, False, "row"),
    (3, 41, 6, 2, 72, 18, "fp32", "fp32", "head", True, True, "far"),
    (2, 33, 8, 2, 128, 64, "bf16", "fp32", "seq", True, False, "far"),
    (2, 33, 8, 2, 128, 64, "bf16", "bf16", "head", False, True, "int32"),
    (1, 19, 5, 5, 80, 20, "fp16", "fp16", "fused", True, False, "back"),
    (2, 9, 2, 1, 256, 128, "bf16", "fp32", "head", True, False, "far"),
    (2, 9, 2, 1, 256, 1, "fp32", "bf16", "head", True, False, "none"),
    (1, 300, 1, 1, 96, 0, "bf16", "fp32", "seq", True, False, "none"),
    (1, 2100, 12, 3, 40, 8, "bf16", "fp32", "seq", True, True, "none"),
    (1, 6, 70, 1, 32, 16, "fp16", "fp32", "seq", False, False, "far"),
]


def _positions(dev, kind, B, N):
    if kind == "none":
        return None
    if kind == "row":
        return torch.arange(5, 5 + N, device=dev)
    if kind == "int32":
        return torch.arange(N, device=dev, dtype=torch.int32).flip(0).expand(B, N)
    if kind == "back":
        return -torch.arange(B * N, device=dev).view(N, B).t()
    return (torch.arange(B, device=dev)[:, None] * 1000003 + (1 << 27) + torch.arange(N, device=dev))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(gpu, case):
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    B, N, H, Hk, D, half, t, wt, layout, norm, inter, pk = case
    q, k, g = _make(gpu, B, N, H, Hk, D, _T[t], layout)
    qw = kw = None
    if norm:
        qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(_T[wt]).to(gpu).requires_grad_(True)
                  for _ in range(2))
    positions = _positions(gpu, pk, B, N)
    freq = _frequencies(half, gpu) if half else None
    eps = 1e-6 if norm else None
    with torch.no_grad():
        plain = qk_norm_rotary(q, k, positions, freq, qw, kw, eps, inter)
    q.requires_grad_(True), k.requires_grad_(True)
    out = qk_norm_rotary(q, k, positions, freq, qw, kw, eps, inter)
    dy = [torch.randn(o.shape, generator=g).to(o.dtype).to(gpu) for o in out]
    leaves = [q, k] + ([qw, kw] if norm else [])
    grads = torch.autograd.grad(out, leaves, dy)
    for a, b in zip(grads, torch.autograd.grad(qk_norm_rotary(q, k, positions, freq, qw, kw, eps, inter),
                                               leaves, dy)):
        assert torch.equal(a, b)
    at = torch.arange(N).expand(B, N) if positions is None else positions.expand(B, N)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        name = "qk"[i]
        assert torch.equal(plain[i], out[i]) and out[i].dtype == x.dtype
        if layout != "fused":
            assert out[i].stride() == x.stride()
        want = _reference(x, dy[i], at, freq, w, eps, inter)
        _check(out[i], want[0], name)
        _check(grads[i], want[1], "d" + name)
        if norm:
            assert grads[2 + i].dtype == w.dtype
            _check(grads[2 + i], want[2], "dw " + name)


def test_against_differences(gpu):
    """Directional differences of the 64-bit formula, FP32 operands."""
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    q, k, g = _make(gpu, 2, 5, 3, 1, 24, torch.float32, "head")
    w = [(1 + 0.3 * torch.randn(24, generator=g)).to(gpu) for _ in range(2)]
    leaves = [t.requires_grad_(True) for t in (q, k, *w)]
    freq = _frequencies(9, gpu)
    out = qk_norm_rotary(*leaves[:2], None, freq, *leaves[2:], 1e-5, True)
    dy = [torch.randn(o.shape, generator=g).to(gpu) for o in out]
    grads = torch.autograd.grad(out, leaves, dy)
    base = [t.detach().double().cpu() for t in leaves]
    at = torch.arange(5).expand(2, 5)

    def loss(ops):
        return sum((_reference(ops[i], None, at, freq, ops[2 + i], 1e-5, True)[0][0]
                    * dy[i].double().cpu()).sum().item() for i in range(2))

    for n, g in enumerate(grads):
        g = g.double().cpu()
        ops = [list(base), list(base)]
        ops[0][n], ops[1][n] = (base[n] + s * 1e-5 * g / g.norm() for s in (1, -1))
        slope = (loss(ops[0]) - loss(ops[1])) / 2e-5
        # The difference's own error: 1e-10 of third derivatives, 2^-53 of the loss / 1e-5.
        assert abs(slope - g.norm().item()) <= 1e-4 * g.norm().item()


def test_broadcast_mixed_and_partial(gpu):
    """Expanded operands, weights of two types, one weight, one output's gradient, more
    than one batch axis and none."""
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    q, k, g = _make(gpu, 6, 7, 4, 2, 32, torch.bfloat16)
    freq = _frequencies(16, gpu).float()
    qw = (1 + 0.3 * torch.randn(32, generator=g)).bfloat16().to(gpu)
    kw = (1 + 0.3 * torch.randn(32, generator=g)).to(gpu)
    want = qk_norm_rotary(q, k, None, freq, qw.float(), kw, 1e-6)
    for a, b in zip(want, qk_norm_rotary(q, k, None, freq, qw, kw, 1e-6)):
        assert torch.equal(a, b)
    many = qk_norm_rotary(*(t.view(2, 3, *t.shape[1:]) for t in (q, k)), torch.arange(7, device=gpu), freq, qw,
                          kw, 1e-6)
    one = qk_norm_rotary(q[4], k[4], torch.arange(7, device=gpu), freq, qw, kw, 1e-6)
    for a, b, c in zip(want, many, one):
        assert torch.equal(a, b.view_as(a)) and torch.equal(a[4], c)
    wide = q[:1, :1].expand(6, 4, 7, 32)
    leaf = q[:1, :1].detach().clone().requires_grad_(True)
    out, _ = qk_norm_rotary(leaf.expand(6, 4, 7, 32), k, None, freq, None, kw, 1e-6)
    assert torch.equal(out, qk_norm_rotary(wide.contiguous(), k, None, freq, None, kw, 1e-6)[0])
    dy = torch.randn(out.shape, generator=g).bfloat16().to(gpu)
    got, = torch.autograd.grad(out, leaf, dy)
    full = wide.contiguous().requires_grad_(True)
    each, = torch.autograd.grad(qk_norm_rotary(full, k, None, freq, None, kw, 1e-6)[0], full, dy)
    sums = each.double().sum((0, 1), keepdim=True)
    assert ((got.double() - sums).abs() <= 2.0 ** -8 * 24 * each.double().abs().sum((0, 1), keepdim=True)).all()


def test_values_that_are_not_finite_stay_in_their_row(gpu):
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    for D, half in ((64, 32), (20, 5)):
        q, k, _ = _make(gpu, 1, 9, 4, 2, D, torch.bfloat16)
        freq = _frequencies(half, gpu)
        clean = qk_norm_rotary(q, k, None, freq, None, None, 1e-6)
        for bad in (float("nan"), float("inf")):
            x = q.clone()
            x[0, 1, 4, 3] = bad
            out, other = qk_norm_rotary(x, k, None, freq, None, None, 1e-6)
            row = torch.zeros(1, 4, 9, dtype=torch.bool, device=gpu)
            row[0, 1, 4] = True
            assert torch.equal(out[~row], clean[0][~row]) and torch.equal(other, clean[1])
            assert not torch.isfinite(out[row]).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,half,t", [(20, 5, "bf16"), (64, 3, "fp32"), (72, 18, "fp16"), (31, 13, "fp32")])
def test_channels_that_pass_stay_apart(gpu, D, half, t, inter):
    """A value that is not finite in a channel that only passes reaches no other channel, in
    the forward, in the backward and on the way into a cache."""
    from openfold3_triangle_kernel_amd import PagedCache, append_kv, qk_norm_rotary

    q, k, g = _make(gpu, 1, 9, 4, 2, D, _T[t])
    freq = _frequencies(half, gpu)
    x = q.clone()
    put = ((2 * half, float("inf")), (2 * half + 3, float("nan")), (D - 1, -float("inf")))
    for c, v in put:
        x[0, :, :, c] = v
    clean, _ = qk_norm_rotary(q, k, None, freq, None, None, None, inter)
    out, _ = qk_norm_rotary(x, k, None, freq, None, None, None, inter)
    assert torch.equal(out[..., :2 * half], clean[..., :2 * half])
    assert torch.equal(out[..., 2 * half:].nan_to_num(9.0), x[..., 2 * half:].nan_to_num(9.0))
    leaf = q.clone().requires_grad_(True)
    turned, _ = qk_norm_rotary(leaf, k, None, freq, None, None, None, inter)
    dx, = torch.autograd.grad(turned, leaf, x, retain_graph=True)
    want, = torch.autograd.grad(turned, leaf, q)
    assert torch.equal(dx[..., :2 * half], want[..., :2 * half])
    assert torch.equal(dx[..., 2 * half:].nan_to_num(9.0), x[..., 2 * half:].nan_to_num(9.0))
    # With a norm an infinity makes its row's other channels 0 and itself NaN.
    x = q.clone()
    x[0, :, :, 2 * half] = float("inf")
    out, _ = qk_norm_rotary(x, k, None, freq, None, None, 1e-6, inter)
    assert out[..., 2 * half].isnan().all()
    out[..., 2 * half] = 0.0
    assert not out.any()
    if D % 8 or t == "fp32":
        return
    cache = PagedCache(2, 2, 16, D, _T[t], gpu)
    starts, lengths, tables = (torch.tensor(n, dtype=torch.int32, device=gpu) for n in ([0, 9], [9], [[1]]))
    x = k[0].transpose(0, 1).clone()
    x[..., 2 * half] = float("inf")
    append_kv(cache, x, x, tables, starts, lengths, None, freq, None, None, None, inter)
    _, want = qk_norm_rotary(q, k, None, freq, None, None, None, inter)
    got = cache.k[1, :, :9]
    assert torch.isposinf(got[..., 2 * half]).all()
    keep = torch.arange(D, device=gpu) != 2 * half
    assert torch.equal(got[..., keep], want[0][..., keep])


def test_zero_heads_and_rows(gpu):
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    freq = _frequencies(8, gpu)
    w = torch.ones(16, device=gpu, requires_grad=True)
    for shape in ((2, 3, 0, 16), (0, 3, 5, 16)):
        q = torch.ones(shape, device=gpu, requires_grad=True)
        out = qk_norm_rotary(q, q, None, freq, w, None, 1e-6)
        assert out[0].shape == shape
        assert not torch.autograd.grad(out[0].sum(), w)[0].any()
    x = torch.zeros(1, 2, 3, 16, device=gpu, requires_grad=True)  # zero rows: the norm's eps alone
    out, _ = qk_norm_rotary(x, x, None, freq, w, None, 1e-6)
    assert not out.any()
    assert torch.isfinite(torch.autograd.grad(out.sum(), x)[0]).all()
    k = torch.randn(1, 2, 3, 16, device=gpu)
    out = qk_norm_rotary(k[:, :0], k, None, freq)
    assert out[0].shape == (1, 0, 3, 16) and torch.equal(out[1], qk_norm_rotary(k, k, None, freq)[0])


def test_another_stream_and_graph(gpu):
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    make = lambda seed: _make(gpu, 2, 50, 8, 2, 64, torch.bfloat16, seed=seed)[:2]  # noqa: E731
    freq = _frequencies(32, gpu)
    w = torch.linspace(0.5, 1.5, 64, device=gpu)
    dy = make(99)

    def step(ops):
        leaves = [t.detach().requires_grad_(True) for t in (*ops, w)]
        out = qk_norm_rotary(*leaves[:2], None, freq, leaves[2], leaves[2], 1e-6)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, dy)]

    want = step(make(0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(make(0))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops = [t.clone() for t in make(0)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step(ops)
    for seed in range(1, 4):
        for t, n in zip(ops, make(seed)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step(make(seed))))


def test_long_operands(gpu):
    """Rows whose byte offsets pass 32 bits."""
    from openfold3_triangle_kernel_amd import qk_norm_rotary

    base = torch.zeros(1400 << 21, device=gpu, dtype=torch.bfloat16)  # 5.9 GB
    q = base.as_strided((1, 1, 1400, 64), (8, 8, 1 << 21, 1))
    q.copy_(torch.randn(1, 1, 1400, 64, generator=torch.Generator().manual_seed(0)).bfloat16())
    freq = _frequencies(32, gpu)
    a = qk_norm_rotary(q, q, None, freq, None, None, 1e-6)[0]
    assert torch.equal(a, qk_norm_rotary(q.contiguous(), q, None, freq, None, None, 1e-6)[0])

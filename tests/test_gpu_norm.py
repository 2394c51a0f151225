"""Layer norm in its types and widths against the formulas in 64 bits.

Tolerances.  Sums over C channels run in chains of at most C / 32 + 32 additions
of 32 bits: t = (C / 32 + 32) 2^-24 relative to the sum of magnitudes.  The mean is
off by t mean|x|, xh = (x - mean) rstd then by e = rstd t mean|x| (1 + |xh|) +
|xh| (t + 2^-21); every further product and sum adds 2^-23 of its operands, the
outputs round once, u = finfo(type).eps / 2.  Column sums run over chains of at
most R / 256 + 64 rows.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(dev, R, C, t, p, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g)) + offset)
    w = 1 + 0.2 * torch.randn(C, generator=g)
    b = 0.2 * torch.randn(C, generator=g)
    dy = torch.randn(R, C, generator=g)
    return (x.to(_T[t]).to(dev), w.to(_T[p]).to(dev), b.to(_T[p]).to(dev), dy.to(_T[t]).to(dev))


def _xh(x, eps=1e-5):
    C = x.shape[-1]
    t = (C / 32 + 32) * 2.0 ** -24
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rstd
    e = rstd * t * x.abs().mean(-1, keepdim=True) * (1 + xh.abs()) + xh.abs() * (t + 2.0 ** -21)
    return xh, rstd, e, t


def _near(got, want, tol, name):
    assert got.shape == want.shape, name
    over = ((got.double().cpu() - want).abs() - tol - 1e-30).max().item()
    assert over <= 0, f"{name}: {over:.3e} over the bound"


def _sub(dtype):  # half the smallest step of the type
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _y_bound(xh, e, w, b, dtype):
    y = xh * w + b
    return y, torch.finfo(dtype).eps / 2 * y.abs() * 1.01 + w.abs() * e + 2.0 ** -22 * (
        (xh * w).abs() + b.abs()) + _sub(dtype)


def _backward_bound(dy, xh, rstd, e, t, w, dtype, pdtype):
    R = dy.shape[0]
    g = dy * w
    m0, m1 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - m0 - xh * m1)
    em1 = (g.abs() * e).mean(-1, keepdim=True) + (t + 2.0 ** -22) * (g * xh).abs().mean(-1, keepdim=True)
    err = rstd * (t * g.abs().mean(-1, keepdim=True) + e * m1.abs() + (xh.abs() + e) * em1
                  + 2.0 ** -21 * (g.abs() + m0.abs() + (xh * m1).abs()))
    erstd = (t + 2.0 ** -21) + rstd * e.amax(-1, keepdim=True) * 0
    err = err + dx.abs() * erstd
    edx = torch.finfo(dtype).eps / 2 * (dx.abs() + err) + err + _sub(dtype)
    chain = (R / 256 + 64) * 2.0 ** -24
    up = torch.finfo(pdtype).eps / 2
    dw, db = (dy * xh).sum(0), dy.sum(0)
    ew = (dy.abs() * e).sum(0) + (chain + 2.0 ** -23) * (dy * xh).abs().sum(0)
    eb = chain * dy.abs().sum(0)
    return (dx, edx), (dw, up * dw.abs() + 1.01 * ew), (db, up * db.abs() + 1.01 * eb)


SHAPES = [  # R, C, rows' type, parameters' type
    (1, 1, "fp32", "fp32"), (3, 7, "bf16", "bf16"), (5, 31, "fp16", "fp32"), (1, 64, "bf16", "fp32"),
    (65, 128, "bf16", "bf16"), (1000, 129, "fp32", "fp32"), (37, 255, "bf16", "fp32"),
    (4, 1024, "bf16", "fp32"), (300, 1000, "fp16", "fp16"), (33, 1531, "fp32", "fp32"),
    (700, 2048, "bf16", "bf16"), (20, 4096, "bf16", "fp32"), (9, 4099, "fp16", "fp16"),
    (6, 8192, "fp32", "fp32"), (3, 8193, "bf16", "bf16"), (5, 20000, "fp32", "bf16"),
    (2, 33333, "bf16", "fp32"),
]


@pytest.mark.parametrize("R,C,t,p", SHAPES, ids=str)
def test_layer_norm(gpu, R, C, t, p):
    from openfold3_triangle_kernel_amd import layer_norm

    x, w, b, dy = _inputs(gpu, R, C, t, p)
    xd, wd, bd, dyd = (v.double().cpu() for v in (x, w, b, dy))
    xh, rstd, e, tt = _xh(xd)
    y, tol = _y_bound(xh, e, wd, bd, x.dtype)
    with torch.no_grad():
        plain = layer_norm(x, w, b)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    out = layer_norm(*leaves)
    assert out.dtype == x.dtype and torch.equal(out, plain)
    _near(out.detach(), y, tol, "y")
    grads = torch.autograd.grad(out, leaves, dy)
    for got, (want, bound), name in zip(grads, _backward_bound(dyd, xh, rstd, e, tt, wd, x.dtype, w.dtype),
                                        ("dx", "dw", "db")):
        _near(got, want, bound, name)
    again = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


def _decode(codes, scales, C):
    k = scales.double() - 127
    v = (codes.double() - 128).reshape(*scales.shape, 32) * torch.exp2(k)[..., None]
    return v.reshape(codes.shape)[:, :C]


@pytest.mark.parametrize("R,C,t,p", SHAPES, ids=str)
def test_layer_norm_int8(gpu, R, C, t, p):
    """The kept codes are within half a step (and xh's own error) of xh, and the
    backward is the formula at the decoded values."""
    from openfold3_triangle_kernel_amd import layer_norm
    from openfold3_triangle_kernel_amd.layernorm import _norm_forward

    x, w, b, dy = _inputs(gpu, R, C, t, p, seed=1)
    xd, wd, bd, dyd = (v.double().cpu() for v in (x, w, b, dy))
    xh, rstd, e, tt = _xh(xd)
    y, _, _, codes, scales = _norm_forward(x, w, b, 1e-5, "int8")
    assert (codes[:, C:] == 128).all()
    kept = _decode(codes.cpu(), scales.cpu(), C)
    step = torch.exp2(scales.cpu().double() - 127).repeat_interleave(32, 1)[:, :C]
    assert ((kept - xh).abs() <= step / 2 + e).all()
    top = (codes.cpu().int() - 128).abs().reshape(R, -1, 32).amax(-1)
    assert ((top <= 127) & ((top >= 63) | (scales.cpu() == 7))).all()
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    out = layer_norm(*leaves, save="int8")
    assert torch.equal(out, y)
    grads = torch.autograd.grad(out, leaves, dy)
    bounds = _backward_bound(dyd, kept, rstd, kept.abs() * 0, tt, wd, x.dtype, w.dtype)
    mean_err = rstd * tt * xd.abs().mean(-1, keepdim=True)  # rstd's error from the mean's
    bounds = ((bounds[0][0], bounds[0][1] + bounds[0][0].abs() * mean_err), *bounds[1:])
    for got, (want, bound), name in zip(grads, bounds, ("dx", "dw", "db")):
        _near(got, want, bound, name)


@pytest.mark.parametrize("save", ["full", "int8"])
def test_parameters_and_views(gpu, save):
    from openfold3_triangle_kernel_amd import layer_norm

    x, w, b, dy = _inputs(gpu, 60, 100, "bf16", "fp32", seed=2)
    want = layer_norm(x, w, b)
    # any leading shape, strided and offset rows
    assert torch.equal(layer_norm(x.view(3, 4, 5, 100), w, b).view(60, 100), want)
    wide = torch.zeros(60, 203, device=gpu, dtype=x.dtype)
    wide[:, 3:103] = x
    strided = wide[:, 3:103]
    assert torch.equal(layer_norm(strided, w, b), want)
    t = x.view(6, 10, 100).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(layer_norm(t, w, b).reshape(60, 100), want)
    leaves = [strided.detach().requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    base = [x.detach().requires_grad_(True), w, b]
    for p, q in zip(torch.autograd.grad(layer_norm(*leaves, save=save), leaves, dy),
                    torch.autograd.grad(layer_norm(*base, save=save), base, dy)):
        assert torch.equal(p, q)
    # a channel-strided input, absent parameters, mixed types, expanded rows
    cs = torch.zeros(60, 200, device=gpu, dtype=x.dtype)
    cs[:, ::2] = x
    assert torch.equal(layer_norm(cs[:, ::2], w, b), want)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    assert torch.equal(layer_norm(x), layer_norm(x, one, zero))
    assert torch.equal(layer_norm(x, w), layer_norm(x, w, zero))
    assert torch.equal(layer_norm(x, None, b), layer_norm(x, one, b))
    assert torch.equal(layer_norm(x, w.bfloat16(), b), layer_norm(x, w.bfloat16().float(), b))
    assert torch.equal(layer_norm(x[:1].expand(60, 100), w, b)[7], want[0])
    for params in ((None, None), (w, None), (None, b), (w.detach(), b), (w, b.detach()),
                   (w.detach().bfloat16().requires_grad_(True), b)):
        xs = x.detach().requires_grad_(True)
        got = [xs, *(q for q in params if q is not None and q.requires_grad)]
        grads = torch.autograd.grad(layer_norm(xs, *params, save=save), got, dy)
        assert all(g.dtype == q.dtype and g.shape == q.shape for g, q in zip(grads, got))
    only = torch.autograd.grad(layer_norm(x.detach(), w, b, save=save), (w, b), dy)
    full = torch.autograd.grad(layer_norm(*base, save=save), base, dy)
    assert torch.equal(only[0], full[1]) and torch.equal(only[1], full[2])


def test_layer_norm_gradient_against_differences(gpu):
    from openfold3_triangle_kernel_amd import layer_norm

    x, w, b, dy = _inputs(gpu, 5, 77, "fp32", "fp32", seed=3)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    base = [v.detach().double().cpu() for v in leaves]

    def loss(ops):
        return ((_xh(ops[0])[0] * ops[1] + ops[2]) * dy.double().cpu()).sum().item()

    for n in range(3):
        g = grads[n].double().cpu()
        d, h = g / g.norm(), 1e-5
        up, down = list(base), list(base)
        up[n], down[n] = base[n] + h * d, base[n] - h * d
        slope = (loss(up) - loss(down)) / (2 * h)
        assert abs(slope - g.norm().item()) <= 1e-5 * g.norm().item()


def test_layer_norm_special_rows(gpu):
    """Constant rows normalise to the bias; a row with NaN is NaN alone, also in the
    gradient from 8 bits."""
    from openfold3_triangle_kernel_amd import layer_norm

    x, w, b, dy = _inputs(gpu, 8, 96, "bf16", "fp32", seed=4)
    x[2] = 3.0
    x[5, 17] = float("nan")
    for save in ("full", "int8"):
        xs = x.detach().requires_grad_(True)
        y = layer_norm(xs, w, b, save=save)
        assert torch.equal(y[2], b.to(y.dtype))
        dx, = torch.autograd.grad(y, xs, dy)
        bad = torch.zeros(8, dtype=torch.bool, device=gpu)
        bad[5] = True
        assert torch.equal(torch.isnan(y).all(-1), bad) and torch.equal(torch.isnan(y).any(-1), bad)
        assert torch.equal(torch.isnan(dx).any(-1), bad) and torch.isfinite(dx[~bad]).all()


@pytest.mark.parametrize("save", ["full", "int8"])
def test_rows_past_32_bits(gpu, save):
    """More than 2^31 elements: a row's results are those of a call on a few rows, the
    parameters' gradients the sums of the parts'."""
    from openfold3_triangle_kernel_amd import layer_norm

    R, C = 2_150_000, 1001
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.empty(R, C, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    dy = torch.empty(R, C, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    w = torch.linspace(0.5, 1.5, C, device=gpu).requires_grad_(True)
    b = torch.zeros(C, device=gpu).requires_grad_(True)

    def run(x, dy):
        xs = x.detach().requires_grad_(True)
        y = layer_norm(xs, w, b, save=save)
        return [y.detach(), *torch.autograd.grad(y, (xs, w, b), dy)]

    whole = run(x, dy)
    for r in (0, 1_072_800, R - 100):
        part = run(x[r:r + 100], dy[r:r + 100])
        assert torch.equal(whole[0][r:r + 100], part[0]) and torch.equal(whole[1][r:r + 100], part[1])
    step = R // 8 + 1
    parts = [run(x[r:r + step], dy[r:r + step])[2:] for r in range(0, R, step)]
    for i in (0, 1):
        total = sum(p[i].double() for p in parts)
        # Chains of R / 512 rows (plus folds) in 32 bits on either side; dy xh is at
        # most of magnitude E|dy xh| < 1 a row.
        assert ((whole[2 + i].double() - total).abs() <= 2 * (R / 512 + 64) * 2.0 ** -24 * R).all()


def test_empty_rows(gpu):
    from openfold3_triangle_kernel_amd import layer_norm

    x = torch.zeros(0, 24, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(24, device=gpu, requires_grad=True)
    y = layer_norm(x, w, None)
    y.sum().backward()
    assert y.shape == (0, 24) and not w.grad.any()


def test_stream_and_graph(gpu):
    from openfold3_triangle_kernel_amd import layer_norm

    x, w, b, dy = _inputs(gpu, 700, 513, "bf16", "fp32", seed=5)

    def step(x, save):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = layer_norm(*leaves, save=save)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    for save in ("full", "int8"):
        want = step(x, save)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(x, save)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        held_x = x.clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            held = step(held_x, save)
        for seed in range(3):
            new = _inputs(gpu, 700, 513, "bf16", "fp32", seed=50 + seed)[0]
            held_x.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(held, step(new, save)))


def test_refusals(gpu):
    from openfold3_triangle_kernel_amd import layer_norm

    x = torch.zeros(4, 16, device=gpu, dtype=torch.bfloat16)
    for args, kw, match in (((x.double(),), {}, "BF16, FP16 or FP32"),
                            ((x.cpu(),), {}, "GPU"),
                            ((x, torch.ones(15, device=gpu)), {}, "shape"),
                            ((x, torch.ones(16)), {}, "device"),
                            ((x, torch.ones(16, device=gpu, dtype=torch.float64)), {}, "FP32"),
                            ((x,), {"save": "int4"}, "save"),
                            ((x,), {"eps": -1.0}, "eps"),
                            ((x[:, :0],), {}, "channels")):
        with pytest.raises(ValueError, match=match):
            layer_norm(*args, **kw)


@pytest.mark.parametrize("save", ["full", "int8"])
@pytest.mark.parametrize("t,wt,bt,size", [("fp32", "fp32", "bf16", 1.0), ("fp32", "fp32", "fp16", 1e6),
                                          ("bf16", "bf16", "fp16", 1e6), ("fp32", "fp16", "bf16", 1.0)])
def test_frozen_weight_beside_a_bias_of_another_type(gpu, save, t, wt, bt, size):
    """The backward uses the weight that the forward used, whatever the type of the
    parameters that want a gradient."""
    from openfold3_triangle_kernel_amd import layer_norm
    from openfold3_triangle_kernel_amd.layernorm import _norm_forward

    x, w, b, dy = _inputs(gpu, 60, 200, t, "fp32", seed=6)
    x.requires_grad_(True)
    w, b = (size * w).to(_T[wt]), b.to(_T[bt]).requires_grad_(True)
    dx, db = torch.autograd.grad(layer_norm(x, w, b, save=save), (x, b), dy)
    xd, wd, dyd = (v.detach().double().cpu() for v in (x, w, dy))
    xh, rstd, e, tt = _xh(xd)
    if save == "int8":
        _, _, _, codes, scales = _norm_forward(x.detach(), None, None, 1e-5, "int8")
        xh, e = _decode(codes.cpu(), scales.cpu(), 200), xh * 0
    (want, tol), _, (wdb, tdb) = _backward_bound(dyd, xh, rstd, e, tt, wd, x.dtype, b.dtype)
    if save == "int8":
        tol = tol + want.abs() * rstd * tt * xd.abs().mean(-1, keepdim=True)  # rstd's, from the mean's
    _near(dx, want, tol, "dx")
    _near(db, wdb, tdb, "db")


@pytest.mark.parametrize("save", ["full", "int8"])
def test_parameter_gradients_of_many_rows(gpu, save):
    """Column sums over 2 150 000 rows against sums in 64 bits, by a bound that a
    workgroup's rows left out would pass.

    Inputs and upstream gradients are independent normal values, so n terms sum to less
    than 6 sqrt(n) in magnitude.  A thread adds n = R / 4096 rows (1024 workgroups of four
    rows), each addition off by at most 2^-24 of the running sum: 2^-24 sum_i 6 sqrt(i) =
    2^-24 4 n^1.5, for 4096 threads; the fold adds 64 + 16 + 4 sums of at most 6 sqrt(R).
    dw also has the error of xh, e a term, which is independent of dy: 6 sqrt(R) e."""
    from openfold3_triangle_kernel_amd import layer_norm
    from openfold3_triangle_kernel_amd.layernorm import _norm_forward

    R, C, u = 2_150_000, 1001, 2.0 ** -24
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.empty(R, C, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    dy = torch.empty(R, C, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    w = torch.ones(C, device=gpu).requires_grad_(True)
    b = torch.zeros(C, device=gpu).requires_grad_(True)
    dw, db = torch.autograd.grad(layer_norm(x, w, b, save=save), (w, b), dy)
    chain = 4096 * u * 4 * (R / 4096) ** 1.5 + u * 6 * R ** 0.5 * (64 + 16 + 4)
    e = 2 * (C / 32 + 32 + 8) * u  # of xh, whose mean square is 1 (|xh| below 6)
    tol_b, tol_w = chain, chain + 6 * R ** 0.5 * 6 * e
    sums = torch.zeros(2, C, device=gpu, dtype=torch.float64)
    share = 4 * -(-R // 4096)  # rows of a workgroup
    step = 25 * share
    for r in range(0, R, step):
        xs, d = x[r:r + step].double(), dy[r:r + step].double()
        if save == "int8":
            _, _, _, codes, scales = _norm_forward(x[r:r + step], None, None, 1e-5, "int8")
            k = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
            xh = ((codes.double() - 128) * k)[:, :C]
        else:
            xh = torch.nn.functional.layer_norm(xs, (C,), eps=1e-5)
        part = torch.stack([(d * xh)[:share].sum(0), d[:share].sum(0)])
        assert part.abs().amax() > tol_w > tol_b  # what a workgroup's rows add is seen
        sums[0] += (d * xh).sum(0)
        sums[1] += d.sum(0)
    assert ((dw.double() - sums[0]).abs() <= tol_w).all()
    assert ((db.double() - sums[1]).abs() <= tol_b).all()

"""Activations in 8 bits: the codec against its rule bit by bit, and the linear layer
that keeps its input so against the formulas in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rule(x, kmax=121):
    """Codes, scales and decoded values of f64 rows, from the rule in 64 bits."""
    R, C = x.shape
    blocks = torch.nn.functional.pad(x, (0, -C % 32)).reshape(R, -1, 32)
    top = blocks.abs().amax(-1)
    finite = torch.isfinite(blocks).all(-1)
    k = torch.full_like(top, -120.0)
    while True:
        more = finite & (torch.round(torch.ldexp(top, -k)) > 127) & (k < kmax)
        if not more.any():
            break
        k = k + more
    q = torch.round(torch.ldexp(blocks, -k[..., None])).clamp(-127, 127)
    q = torch.where(finite[..., None], q, 0.0)
    values = torch.where(finite[..., None], torch.ldexp(q, k[..., None]), float("nan"))
    scales = torch.where(finite, k + 127, 255.0)
    return (q + 128).reshape(R, -1), scales, values.reshape(R, -1)[:, :C]


@pytest.mark.parametrize("t", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 31), (2, 32), (7, 100), (129, 257), (1000, 64), (5, 5001)])
def test_codec(gpu, R, C, t):
    from openfold3_triangle_kernel_amd import compress_activation, decompress_activation

    g = torch.Generator().manual_seed(R + C)
    x = torch.randn(R, C, generator=g) * torch.exp2(
        torch.randint(-12, 12, (R, C), generator=g).float() * (torch.rand(R, C, generator=g) < 0.1))
    x = x.to(_T[t])
    saved = compress_activation(x.to(gpu))
    codes, scales, values = _rule(x.double())
    assert torch.equal(saved.codes.cpu().double(), codes)
    assert torch.equal(saved.scales.cpu().double(), scales)
    assert saved.nbytes == codes.numel() + scales.numel()
    back = decompress_activation(saved)
    assert back.dtype == x.dtype and back.shape == x.shape
    assert torch.equal(back.cpu(), values.to(x.dtype))
    assert torch.equal(decompress_activation(saved, torch.float32).cpu().double(), values)
    top = torch.nn.functional.pad(x.double(), (0, -C % 32)).reshape(R, -1, 32).abs().amax(-1)
    # The largest is at least 63.75 steps (127.5 of the step below would round to
    # 128), so half a step is at most its 1/127.5.
    err = (values - x.double()).abs()
    assert (err <= top.repeat_interleave(32, 1)[:, :C] / 127.5).all()


def test_codec_edges(gpu):
    """Ties, the border at 127.5, zeros, the range's ends, infinities and NaN."""
    from openfold3_triangle_kernel_amd import compress_activation, decompress_activation

    rows = torch.zeros(12, 64)
    rows[0, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5])
    rows[1, :3] = torch.tensor([127.5, 1.0, 3.0])
    rows[2, :3] = torch.tensor([127.49, 1.0, 0.5])
    rows[3, 0] = 2.0 ** 127
    rows[4, 0] = torch.finfo(torch.float32).max
    rows[5, :2] = torch.tensor([2.0 ** -120, 2.0 ** -121])
    rows[6, :2] = torch.tensor([2.0 ** -126, 1e-44])
    rows[7, 5] = float("inf")
    rows[8, 40] = float("nan")
    rows[9, 3] = float("-inf")
    rows[10, :2] = torch.tensor([-0.0, 63.75])
    rows[11, :2] = torch.tensor([-torch.finfo(torch.float32).max, 2.0 ** 121])
    saved = compress_activation(rows.to(gpu))
    codes, scales, values = _rule(rows.double())
    assert torch.equal(saved.codes.cpu().double(), codes)
    assert torch.equal(saved.scales.cpu().double(), scales)
    back = decompress_activation(saved).cpu()
    assert torch.equal(torch.isnan(back), torch.isnan(values))
    assert torch.equal(back[~torch.isnan(back)].double(), values[~torch.isnan(values)])
    assert torch.isnan(back[7, :32]).all() and not back[7, 32:].any()
    assert torch.isfinite(back[[3, 4, 11]]).all()
    half = torch.zeros(3, 32, dtype=torch.float16)
    half[0, :2] = torch.tensor([65504.0, -300.0])
    half[1, :2] = torch.tensor([-65280.0, 256.0])
    half[2, 0] = 65279.0
    saved = compress_activation(half.to(gpu))
    codes, scales, values = _rule(half.double(), 9)
    assert torch.equal(saved.codes.cpu().double(), codes)
    assert torch.equal(saved.scales.cpu().double(), scales)
    assert torch.equal(decompress_activation(saved).cpu().double(), values)
    assert torch.isfinite(values).all() and (values - half.double()).abs().max() <= 65504 / 127.5


def test_codec_views_and_empty(gpu):
    from openfold3_triangle_kernel_amd import compress_activation, decompress_activation

    x = torch.randn(4, 6, 75, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    want = decompress_activation(compress_activation(x))
    wide = torch.zeros(4, 6, 81, device=gpu, dtype=x.dtype)
    wide[..., 5:80] = x
    assert torch.equal(decompress_activation(compress_activation(wide[..., 5:80])), want)
    t = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(decompress_activation(compress_activation(t)), want)
    none = decompress_activation(compress_activation(x[:0]))
    assert none.shape == (0, 6, 75)
    assert not compress_activation(x.float().requires_grad_(True)).codes.requires_grad


CASES = [  # R, K, N, weight's type
    (1, 8, 8, "bf16"), (3, 32, 16, "fp32"), (63, 40, 136, "bf16"), (257, 128, 512, "bf16"),
    (1000, 136, 72, "fp32"), (700, 512, 128, "bf16"), (2049, 264, 392, "bf16"), (9000, 128, 64, "fp32"),
]


@pytest.mark.parametrize("save", ["int8", "full"])
@pytest.mark.parametrize("R,K,N,t", CASES, ids=str)
def test_linear(gpu, R, K, N, t, save):
    """Products of BF16 operands sum in 32 bits: chains of at most n / 8 + 300
    additions of 2^-24 relative to the sum of magnitudes (n the summed axis), and one
    rounding of the output, 2^-8 for BF16."""
    from openfold3_triangle_kernel_amd import linear

    g = torch.Generator().manual_seed(R)
    x = torch.randn(R, K, generator=g).bfloat16()
    w = (torch.randn(N, K, generator=g) / K ** 0.5).to(_T[t])
    dy = torch.randn(R, N, generator=g).bfloat16()
    leaves = [v.to(gpu).requires_grad_(True) for v in (x, w)]
    y = linear(*leaves, save=save)
    dx, dw = torch.autograd.grad(y, leaves, dy.to(gpu))
    xd, wd, dyd = x.double(), w.bfloat16().double(), dy.double()
    kept = _rule(xd)[2] if save == "int8" else xd

    def check(got, a, b, dtype, name):
        want = a @ b
        n = a.shape[1]
        tol = 2.0 ** -24 * (n / 8 + 300) * (a.abs() @ b.abs())
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
        assert got.dtype == dtype, name
        over = ((got.double().cpu() - want).abs() - tol - 1e-30).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"

    check(y.detach(), xd, wd.t(), torch.bfloat16, "y")
    check(dx, dyd, wd, torch.bfloat16, "dx")
    check(dw, dyd.t(), kept, w.dtype, "dw")
    again = torch.autograd.grad(linear(*leaves, save=save), leaves, dy.to(gpu))
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_linear_views(gpu):
    from openfold3_triangle_kernel_amd import linear

    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 25, 64, generator=g).bfloat16().to(gpu)
    w = torch.randn(48, 64, generator=g).bfloat16().to(gpu)
    dy = torch.randn(4, 25, 48, generator=g).bfloat16().to(gpu)

    def grads(x, w, dy):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = linear(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)]

    want = grads(x, w, dy)
    wide = torch.zeros(4, 25, 75, device=gpu, dtype=x.dtype)
    wide[..., 3:67] = x
    t = x.transpose(0, 1).contiguous().transpose(0, 1)
    wt = w.t().contiguous().t()
    for a, b, c in ((wide[..., 3:67], w, dy), (t, wt, dy), (x, w, dy.float().double()),
                    (x, w, dy.transpose(0, 1).contiguous().transpose(0, 1))):
        c = c.to(torch.bfloat16) if c.dtype == torch.float64 else c
        assert all(torch.equal(p, q) for p, q in zip(grads(a, b, c), want))
    assert torch.equal(linear(x.view(100, 64), w).view(4, 25, 48), want[0])
    ones = torch.autograd.grad(linear(x, w.requires_grad_(True)).sum(), w)[0]  # expanded dy
    assert torch.equal(ones, grads(x, w, torch.ones_like(dy))[2])
    empty = linear(x[:0].requires_grad_(True), w)
    empty.sum().backward()
    assert empty.shape == (0, 25, 48) and not w.grad.any()


def test_rows_past_32_bits(gpu):
    """dy and the codec's rows beyond 2^31 elements (and 4 GiB): rows are those of a call
    on a few of them, the weight's gradient the sum of the parts'."""
    from openfold3_triangle_kernel_amd import compress_activation, decompress_activation, linear

    R, K, N = 4_250_000, 24, 512
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.empty(R, K, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    w = torch.empty(N, K, device=gpu, dtype=torch.bfloat16).normal_(generator=g).requires_grad_(True)
    dy = torch.empty(R, N, device=gpu, dtype=torch.bfloat16).normal_(generator=g)

    def run(x, dy):
        xs = x.detach().requires_grad_(True)
        y = linear(xs, w)
        return [y.detach(), *torch.autograd.grad(y, (xs, w), dy)]

    whole = run(x, dy)
    for r in (0, 2_096_900, 4_194_200, R - 100):
        part = run(x[r:r + 100], dy[r:r + 100])
        assert torch.equal(whole[0][r:r + 100], part[0]) and torch.equal(whole[1][r:r + 100], part[1])
    step = R // 8 + 1
    total = sum(run(x[r:r + step], dy[r:r + step])[2].double() for r in range(0, R, step))
    # Nine roundings to BF16 of parts no larger than their magnitudes' sum.
    assert ((whole[2].double() - total).abs() <= 9 * 2.0 ** -8 * 5 * R ** 0.5).all()
    saved = compress_activation(dy)
    for r in (0, 2_096_900, 4_194_200, R - 100):
        few = compress_activation(dy[r:r + 100])
        assert torch.equal(saved.codes[r:r + 100], few.codes)
        assert torch.equal(saved.scales[r:r + 100], few.scales)
    back = decompress_activation(saved)
    assert torch.equal(back[-100:], decompress_activation(few))


def test_stream_and_graph(gpu):
    from openfold3_triangle_kernel_amd import compress_activation, decompress_activation, linear

    g = torch.Generator().manual_seed(3)
    x = torch.randn(3000, 96, generator=g).bfloat16().to(gpu)
    w = torch.randn(64, 96, generator=g).bfloat16().to(gpu)
    dy = torch.randn(3000, 64, generator=g).bfloat16().to(gpu)

    def step(x):
        leaves = [t.detach().requires_grad_(True) for t in (x, w)]
        y = linear(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy),
                decompress_activation(compress_activation(x))]

    held_x = x.clone()
    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step(held_x)
    for seed in range(3):
        new = torch.randn(3000, 96, generator=g).bfloat16().to(gpu)
        held_x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step(new)))


@pytest.mark.parametrize("save", ["int8", "full"])
def test_linear_of_far_rows(gpu, save):
    """Rows further apart than the GEMM's 32-bit offsets serve, in the input and in the
    gradient: as of their contiguous copies."""
    from openfold3_triangle_kernel_amd import linear

    g = torch.Generator().manual_seed(5)
    far = torch.zeros(3, (1 << 24) + 8, device=gpu, dtype=torch.bfloat16)
    x, dy = far[:, :64], far[:, 64:64 + 24]
    x.copy_(torch.randn(3, 64, generator=g))
    dy.copy_(torch.randn(3, 24, generator=g))
    runs = []
    for rows, grad in ((x, dy), (x.contiguous(), dy.contiguous())):
        rows = rows.detach().requires_grad_(True)
        w = torch.randn(24, 64, generator=torch.Generator().manual_seed(6)).to(gpu).requires_grad_(True)
        y = linear(rows, w, save=save)
        runs.append((y, *torch.autograd.grad(y, (rows, w), grad)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_refusals(gpu):
    from openfold3_triangle_kernel_amd import compress_activation, decompress_activation, linear

    x = torch.zeros(4, 16, device=gpu, dtype=torch.bfloat16)
    w = torch.zeros(8, 16, device=gpu, dtype=torch.bfloat16)
    big = torch.zeros((1 << 23) + 8, 8, device=gpu, dtype=torch.bfloat16)
    for call, match in ((lambda: compress_activation(x.cpu()), "GPU"),
                        (lambda: compress_activation(x.double()), "BF16"),
                        (lambda: compress_activation(x[:, :0]), "channels"),
                        (lambda: decompress_activation(x), "CompressedActivation"),
                        (lambda: decompress_activation(compress_activation(x), torch.int8), "gives"),
                        (lambda: linear(x.float(), w), "BF16 input"),
                        (lambda: linear(x, w[:, :8]), "weight"),
                        (lambda: linear(x, w[:4]), "multiples of 8"),
                        (lambda: linear(x[:, :12], w[:, :12]), "multiples of 8"),
                        (lambda: linear(x[:, :8], big), "2\\^23"),
                        (lambda: linear(x, w.cpu()), "device"),
                        (lambda: linear(x, w.half()), "weight"),
                        (lambda: linear(x, w, save="none"), "save")):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("save", ["int8", "full"])
def test_weight_gradient_of_rows_past_2_gib(gpu, save):
    """dy beyond 2 GiB: both modes give the sum of the parts' gradients, in 32 bits.

    With an FP32 weight either side is a sum in 32 bits of products exact in it.  Terms are
    independent of mean 0 (x and dy normal), so n of them sum to less than 6 sqrt(n) in
    magnitude.  A split (128 of them) adds its R / 128 rows 16 at a time, two roundings of
    the running sum a time: 2^-23 sum_i 6 sqrt(16 i) = 2^-23 16 (R / 2048)^1.5; the folds add
    300 sums of at most 6 sqrt(R).  The parts' own splits are shorter."""
    from openfold3_triangle_kernel_amd import linear

    R, K, N = 4_250_000, 24, 512
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.empty(R, K, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    dy = torch.empty(R, N, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    w = torch.empty(N, K, device=gpu).normal_(generator=g).requires_grad_(True)

    def grad(x, dy):
        return torch.autograd.grad(linear(x, w, save=save), w, dy)[0]

    whole = grad(x, dy)
    step = R // 8 + 1
    total = sum(grad(x[r:r + step], dy[r:r + step]).double() for r in range(0, R, step))
    bound = 2 * (128 * 2.0 ** -23 * 16 * (R / 2048) ** 1.5 + 300 * 2.0 ** -24 * 6 * R ** 0.5)
    assert bound < 0.3 * (R / 128) ** 0.5  # a split's rows left out would show
    assert ((whole.double() - total).abs() <= bound).all()


@pytest.mark.parametrize("save", ["int8", "full"])
@pytest.mark.parametrize("pitch", [64, 75, 72, (1 << 24) + 8])
def test_linear_of_one_row(gpu, save, pitch):
    """A single row's stride addresses nothing and may be anything, in the input and in
    the gradient."""
    from openfold3_triangle_kernel_amd import linear

    g = torch.Generator().manual_seed(7)
    wide = torch.zeros(pitch, device=gpu, dtype=torch.bfloat16)
    x, dy = wide.as_strided((1, 64), (pitch, 1)), wide.clone().as_strided((1, 24), (pitch, 1))
    x.copy_(torch.randn(1, 64, generator=g))
    dy.copy_(torch.randn(1, 24, generator=g))
    runs = []
    for rows, grad in ((x, dy), (x.clone().contiguous(), dy.clone().contiguous())):
        rows = rows.detach().requires_grad_(True)
        w = torch.randn(24, 64, generator=torch.Generator().manual_seed(8)).to(gpu).requires_grad_(True)
        y = linear(rows, w, save=save)
        runs.append((y, *torch.autograd.grad(y, (rows, w), grad)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))

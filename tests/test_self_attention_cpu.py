"""Refusals of self-attention's operators without a GPU: host tensors and bad arguments
raise before any native call, the C ABI answers bad shapes with a status before any
launch, and the rule of a paged cache's places on host arrays."""

import ctypes

import pytest
import torch

from openfold3_triangle_kernel_amd import (PagedCache, _native, append_kv, paged_attention, qk_norm_rotary,
                                           window_attention)
from openfold3_triangle_kernel_amd.paged import batch_struct


def _qk(B=1, H=2, Hk=2, N=4, D=16, dtype=torch.bfloat16):
    return torch.zeros(B, H, N, D, dtype=dtype), torch.zeros(B, Hk, N, D, dtype=dtype)


_F = torch.ones(8)


@pytest.mark.parametrize("args,match", [
    ((*_qk(),), "GPU"),
    ((_qk()[0], None), "torch.Tensor"),
    ((*(t[0, 0] for t in _qk()),), "shape"),
    ((*_qk(dtype=torch.float64),), "BF16, FP16 or FP32"),
    ((_qk()[0], _qk(dtype=torch.float16)[1]), "share one type"),
    ((_qk(N=5)[0], _qk()[1]), "positions"),
    ((_qk(B=2)[0], _qk()[1]), "prefix"),
    ((*_qk(D=257),), "D<=256"),
    ((*_qk(), torch.zeros(4)), "int32 or int64"),
    ((*_qk(), torch.zeros(3, dtype=torch.int64)), "broadcast"),
    ((*_qk(), torch.zeros(2, 4, dtype=torch.int64)), "broadcast"),
    ((*_qk(), None, torch.ones(9)), "more pairs"),
    ((*_qk(), None, torch.ones(8, dtype=torch.int64)), "floating"),
    ((*_qk(), None, torch.ones(2, 4)), "one axis"),
    ((*_qk(), None, torch.ones(8, requires_grad=True)), "must not require"),
    ((*_qk(), None, _F, torch.ones(16)), "give eps"),
    ((*_qk(), None, _F, torch.ones(15), None, 1e-6), "shape"),
    ((*_qk(), None, _F, torch.ones(16, dtype=torch.float64), None, 1e-6), "BF16, FP16 or FP32"),
    ((*_qk(), None, _F, None, None, -1e-6), "eps"),
    ((*_qk(), None, _F, None, None, float("nan")), "eps"),
])
def test_rotary_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        qk_norm_rotary(*args)


def _paged(S=2, T=3, Hk=2, D=16, width=2, page=4, pages=5):
    cache = PagedCache(pages, Hk, page, D, device="cpu")
    tables = torch.zeros(S, width, dtype=torch.int32)
    starts, lengths = torch.zeros(S + 1, dtype=torch.int32), torch.zeros(S, dtype=torch.int32)
    return cache, torch.zeros(T, Hk, D).bfloat16(), tables, starts, lengths


def test_cache_refuses():
    good = torch.zeros(3, 2, 4, 16).bfloat16()
    for k, v, match in ((good, good[:2], "alike"), (good.float(), good.float(), "BF16 or FP16"),
                        (good[0], good[0], r"\[pages"), (good, good.half(), "alike"),
                        (good[..., :12], good[..., :12], "contiguous"),
                        (good[..., :4].contiguous(), good[..., :4].contiguous(), "multiple of 8"),
                        (None, good, r"\[pages"),
                        (good.clone().requires_grad_(True), good, "gradients")):
        with pytest.raises(ValueError, match=match):
            PagedCache.of(k, v)
    with pytest.raises(ValueError, match="multiple of 8"):
        PagedCache(3, 2, 4, 136, device="cpu")
    cache = PagedCache.of(good, good)
    assert (cache.pages, cache.kv_heads, cache.page, cache.head_dim) == (3, 2, 4, 16)


def test_append_refuses():
    cache, x, tables, starts, lengths = _paged()
    cases = [((cache, x, x, tables, starts, lengths), "GPU"),
             ((None, x, x, tables, starts, lengths), "PagedCache"),
             ((cache, x, x, tables.long(), starts, lengths), "int32"),
             ((cache, x, x, tables[0], starts, lengths), "2 axes"),
             ((cache, x, x, tables, starts[:2], lengths), "S, S"),
             ((cache, x, x, tables[:1], starts, lengths), "S, S"),
             ((cache, x, x, tables.t().contiguous().t(), starts, lengths), "contiguous"),
             ((cache, x[:, :1], x, tables, starts, lengths), "kv heads"),
             ((cache, x, x[:2], tables, starts, lengths), "shape"),
             ((cache, x, x.half(), tables, starts, lengths), "type"),
             ((cache, x[..., :8], x, tables, starts, lengths), "shape"),
             ((cache, x, x, tables, starts, lengths, x[0]), "shape"),
             ((cache, x.clone().requires_grad_(True), x, tables, starts, lengths), "no_grad"),
             ((cache, x, x, tables, starts, lengths, None, torch.ones(9)), "more pairs"),
             ((cache, x, x, tables, starts, lengths, None, None, torch.ones(16)), "give eps"),
             ((cache, x, x, torch.zeros(2, 1 << 29, dtype=torch.int32), starts, lengths), "2\\^30")]
    for args, match in cases:
        with pytest.raises(ValueError, match=match):
            append_kv(*args)


def test_places_of_a_cache():
    """``tpf_paged_row`` on host arrays: the rule that the kernels share."""
    cache, _, tables, starts, lengths = _paged(S=3, width=3, page=4, pages=7)
    tables.copy_(torch.tensor([[6, 0, 3], [7, -1, 2], [1, 2 ** 31 - 1, 5]]))
    batch = batch_struct(cache.k, tables, starts, lengths, 5)
    row = lambda s, j: _native.query("tpf_paged_row", ctypes.byref(batch), s, j)  # noqa: E731
    for s in range(3):
        for j in range(12):
            p = int(tables[s, j // 4])
            assert row(s, j) == (p * 4 + j % 4 if 0 <= p < 7 else -1)
        assert row(s, -1) == row(s, 12) == row(s, 1 << 40) == -1
    assert row(3, 0) == row(-1, 0) == -1


@pytest.mark.parametrize("S,T,G", [(3, 200, 4), (3, 1000, 4), (4, 300, 1), (70, 900, 3), (70, 5000, 8),
                                   (200, 777, 40), (1, 65, 7)])
def test_rows_of_a_batch(S, T, G):
    """``tpf_paged_rows``, the rule by which the attention finds the rows of its tiles and of
    its join: ascending starts give every row once, any others rows of the batch alone."""
    cache, _, tables, starts, lengths = _paged(S=S)
    batch = batch_struct(cache.k, tables, starts, lengths, T)
    out = (ctypes.c_int64 * 3)()

    def rows(tile_rows, at):
        """(first row, all rows of its sequence, the sequence's first row in the batch)."""
        if _native.query("tpf_paged_rows", ctypes.byref(batch), G, tile_rows, at, out) < 0:
            return None
        first, count, token = out
        assert 0 <= first < count and 0 <= token and token * G + count <= T * G, (tile_rows, at, *out)
        return first, count, token * G

    def check(ascending):
        for tile_rows in (32, 128):
            met = torch.zeros(T * G, dtype=torch.int32)
            for at in range(T * G // tile_rows + S + 1):
                got = rows(tile_rows, at)
                if got:
                    first, count, base = got
                    met[base + first:base + min(first + tile_rows, count)] += 1
            assert not ascending or (met == 1).all()
        for at in range(0, T * G, max(1, T * G // 500)):
            got = rows(0, at)
            assert got[0] + got[2] == at if got else not ascending

    g = torch.Generator().manual_seed(S * T + G)
    draw = lambda low, high: torch.randint(low, high, (S + 1,), generator=g, dtype=torch.int32)  # noqa: E731
    for _ in range(4):
        starts.copy_(draw(0, T + 1).sort()[0])
        starts[0] = 0
        check(True)
        starts.copy_(draw(-T, 2 * T))
        check(False)
        starts.copy_(draw(0, T + 1).sort(descending=True)[0])
        check(False)
        starts.copy_(draw(0, T + 1).sort()[0])
        starts[S // 2 + 1:] = 0  # (a batch's rows, then what a padded graph's array holds)
        check(False)
    for bad in ((0, 32, 0), (G, 64, 0), (G, 32, -1), (G, 32, T * G // 32 + S + 1), (G, 0, T * G), (1 << 30, 32, 0)):
        assert _native.query("tpf_paged_rows", ctypes.byref(batch), *bad, out) == -1


def test_c_abi_answers_before_a_launch():
    shape = (ctypes.c_int64 * 25)(1, 4, 2, 2, 16, 9, 0, 2, 1, 0, 64)
    with pytest.raises(RuntimeError, match="half=9"):
        _native.call("tpf_rotary_forward", 16, 16, None, 16, None, None, 1e-6, 16, 16, shape, None)
    shape[5] = 8
    with pytest.raises(RuntimeError, match="null pointer"):
        _native.call("tpf_rotary_forward", 16, 16, None, None, None, None, 1e-6, 16, 16, shape, None)
    with pytest.raises(RuntimeError, match="eps"):
        _native.call("tpf_rotary_forward", 16, 16, None, 16, None, None, -1.0, 16, 16, shape, None)
    shape[10] = 16
    with pytest.raises(RuntimeError, match="32 or 64"):
        _native.call("tpf_rotary_forward", 16, 16, None, 16, None, None, 1e-6, 16, 16, shape, None)
    shape[10] = 64
    with pytest.raises(RuntimeError, match="workspace"):
        _native.call("tpf_rotary_backward", 16, 16, 16, 16, None, 16, 16, 16, 1e-6, 16, 16, 16, 16,
                     16, 8, shape, (ctypes.c_int64 * 6)(), None)
    assert _native.query("tpf_rotary_backward_workspace_bytes", shape) == 1 * 2 * 16 * 4
    shape[4] = 257
    assert _native.query("tpf_rotary_backward_workspace_bytes", shape) == -1
    cache, x, tables, starts, lengths = _paged()
    batch = batch_struct(cache.k, tables, starts, lengths, 3)
    append = (ctypes.c_int64 * 14)(0, 2, 16, 0, 2, 2)
    with pytest.raises(RuntimeError, match="TPF_BF16 or TPF_F16"):
        _native.call("tpf_paged_append", None, 16, 16, None, None, None, 0.0, None, 16, 16, append,
                     ctypes.byref(batch), None)
    batch.page = 0
    with pytest.raises(RuntimeError, match="bad batch"):
        _native.call("tpf_paged_append", None, 16, 16, None, None, None, 0.0, None, 16, 16, append,
                     ctypes.byref(batch), None)


def _qkv(B=1, H=2, Hk=2, N=4, D=64, dtype=torch.bfloat16):
    return [torch.zeros(B, h, N, D, dtype=dtype) for h in (H, Hk, Hk)]


@pytest.mark.parametrize("args,match", [
    ((*_qkv(),), "GPU"),
    ((_qkv()[0], _qkv()[1], None), "torch.Tensor"),
    ((*(t[0, 0] for t in _qkv()),), "shape"),
    ((*_qkv(dtype=torch.float32),), "BF16 or FP16"),
    ((*_qkv(D=129),), "D<=128"),
    ((*_qkv(H=3),), "multiple"),
    ((_qkv()[0], _qkv()[1], _qkv(N=5)[2]), "one shape"),
    ((_qkv(N=5)[0], *_qkv()[1:]), "tokens"),
    ((_qkv(B=2)[0], *_qkv()[1:]), "batch prefix"),
    ((*_qkv(), 0), "window"),
    ((*_qkv(), 2.0), "window"),
    ((*_qkv(), 2, -1), "sinks"),
    ((*_qkv(), 2, None), "sinks"),
    ((*_qkv(), 2, 1, torch.zeros(4)), "boolean"),
    ((*_qkv(), 2, 1, torch.zeros(3, dtype=torch.bool)), "broadcast"),
    ((*_qkv(), 2, 1, torch.zeros(2, 4, dtype=torch.bool)), "broadcast"),
    ((*_qkv(), 2, 1, torch.zeros(1, dtype=torch.bool)), "broadcast"),
    ((*_qkv(), None, 0, None, 0.0), "scale"),
    ((*_qkv(), None, 0, None, float("nan")), "scale"),
])
def test_window_attention_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        window_attention(*args)


def test_paged_attention_refuses():
    cache, x, tables, starts, lengths = _paged()
    q = torch.zeros(3, 4, 16).bfloat16()
    for args, match in (((q, cache, tables, starts, lengths), "GPU"),
                        ((q, None, tables, starts, lengths), "PagedCache"),
                        ((q[:, :3], cache, tables, starts, lengths), "multiple"),
                        ((q[:, :0], cache, tables, starts, lengths), "multiple"),
                        ((q[0], cache, tables, starts, lengths), "shape"),
                        ((q.half(), cache, tables, starts, lengths), "type"),
                        ((q, cache, tables.long(), starts, lengths), "int32"),
                        ((q, cache, tables, starts, lengths[:1]), "S, S"),
                        ((q.clone().requires_grad_(True), cache, tables, starts, lengths), "no_grad"),
                        ((q, cache, tables, starts, lengths, 0), "window"),
                        ((q, cache, tables, starts, lengths, 4, -1), "sinks"),
                        ((q, cache, tables, starts, lengths, 4, 1, -1.0), "scale")):
        with pytest.raises(ValueError, match=match):
            paged_attention(*args)


def test_attention_c_abi_answers_before_a_launch():
    shape = (ctypes.c_int64 * 18)(1, 4, 2, 100, 64, 0, 10, 2, 0)
    q = lambda name, *args: _native.query(name, *args)  # noqa: E731
    assert q("tpf_window_forward_workspace_bytes", shape) == 0
    assert q("tpf_window_backward_workspace_bytes", shape) == 4 * 100 * 4
    call = lambda s=shape, fn="tpf_window_forward": _native.call(  # noqa: E731
        fn, *([16] * (4 if fn == "tpf_window_forward" else 12)), *(
            [16, None, None, None, 0] if fn == "tpf_window_forward" else [8]), s, *(
            [] if fn == "tpf_window_forward" else [(ctypes.c_int64 * 9)()]), 0.125, None)
    for at, value, match in ((1, 3, "H=3"), (4, 136, "D=136"), (4, 12, "D=12"), (3, 0, "rows"),
                             (3, 1 << 40, "rows"), (5, 2, "TPF_BF16"), (6, -1, "window"), (7, -1, "window"),
                             (9, 4, "multiples of 8"), (14, 1 << 23, "state stride")):
        bad = (ctypes.c_int64 * 18)(*shape)
        bad[at] = value
        with pytest.raises(RuntimeError, match=match):
            call(bad)
        assert q("tpf_window_forward_workspace_bytes", bad) == -1
    with pytest.raises(RuntimeError, match="workspace"):
        call(fn="tpf_window_backward_bf16")
    cache, x, tables, starts, lengths = _paged()
    batch = batch_struct(cache.k, tables, starts, lengths, 3)
    paged = (ctypes.c_int64 * 8)(4, 2, 16, 0, 0, 0, 64, 16)
    size = lambda s=paged: q("tpf_paged_attention_workspace_bytes", s, ctypes.byref(batch))  # noqa: E731
    assert size() == 0
    batch.width, batch.page, batch.pages = 64, 64, 100
    assert size() > 0
    for at, value in ((0, 3), (2, 12), (3, 2), (4, -1), (5, -1), (6, 4)):
        bad = (ctypes.c_int64 * 8)(*paged)
        bad[at] = value
        assert size(bad) == -1
    batch.pages = 1 << 25
    assert size() == -1


def test_block_on_the_cpu():
    """The block's formulas in PyTorch: masks, windows, empty rows, the routing policy."""
    from openfold3_triangle_kernel_amd import (SelfAttention, set_turbopairformer_strict,
                                               stock_invocation_count)

    torch.manual_seed(0)
    block = SelfAttention(24, 8, 4, 2, window=3, sinks=1)
    x = torch.randn(2, 6, 24, requires_grad=True)
    before = stock_invocation_count()
    out = block(x)
    assert stock_invocation_count() == before + 1 and out.shape == x.shape
    # A token that nothing later sees changes nothing later; all see the first one.
    for at, seen_by in ((0, range(6)), (2, (2, 3, 4)), (5, (5,))):
        other = x.detach().clone()
        other[:, at, :12] += 1.0  # (the norm takes out what all channels share)
        changed = (block(other) - out).abs().amax((0, 2)) > 1e-6
        assert changed.tolist() == [i in seen_by for i in range(6)]
    mask = torch.ones(2, 6, dtype=torch.bool)
    mask[1, :4] = False
    masked = block(x, mask)
    assert torch.equal(masked[0], out[0]) and not masked[1, :4].any()
    g, = torch.autograd.grad(masked.sum(), x)
    assert torch.isfinite(g).all() and not g[1, :4].any()
    assert block(x[:, :0]).shape == (2, 0, 24)
    far = block(x, positions=torch.arange(6) + 1000)  # rotations are relative
    assert (far - out).abs().max() <= 1e-4
    wide = SelfAttention(24, 8, 4, 2, frequencies=block._frequencies["cpu"], window=3, sinks=1)
    wide.load_state_dict(block.state_dict())
    assert torch.equal(wide(x), out)
    set_turbopairformer_strict(True)
    try:
        with pytest.raises(RuntimeError, match="strict"):
            block(x)
    finally:
        set_turbopairformer_strict(False)
    with pytest.raises(ValueError, match="BF16"):
        block.step(x[0], None, None, None, None)
    for bad in (dict(no_heads=3, no_kv_heads=2), dict(no_heads=2, activation_save="int4"),
                dict(no_heads=2, window=0), dict(no_heads=2, sinks=-1), dict(no_heads=2, rotary_channels=3),
                dict(no_heads=2, rotary_channels=10), dict(no_heads=2, frequencies=torch.ones(5))):
        with pytest.raises(ValueError):
            SelfAttention(8, 8, **bad)


@pytest.fixture
def fake(monkeypatch):
    """The facades on host tensors, the native calls recorded instead of made."""
    import sys

    calls = []
    monkeypatch.setattr(_native, "call", lambda name, *args: calls.append(name))
    monkeypatch.setattr(_native, "query", lambda name, *args: 0)
    for name in ("rotary", "window_attention", "paged"):
        monkeypatch.setattr(sys.modules[f"openfold3_triangle_kernel_amd.{name}"], "_device_supported",
                            lambda t: (True, ""))
    return calls


def _calls():
    g = torch.Generator().manual_seed(0)
    draw = lambda *shape: torch.randn(*shape, generator=g).bfloat16()  # noqa: E731
    cache, x, tables, starts, lengths = _paged()
    places = (tables, starts, lengths)
    return {"rotary": (lambda q, k, w: qk_norm_rotary(q, k, None, _F, w, w, 1e-6),
                       (draw(1, 2, 4, 16), draw(1, 2, 4, 16), draw(16))),
            "window": (lambda q, k, v: window_attention(q, k, v, 3, 1),
                       (draw(1, 2, 4, 16), draw(1, 2, 4, 16), draw(1, 2, 4, 16))),
            "append": (lambda k, v, q: append_kv(cache, k, v, *places, q, _F), (x, x.clone(), draw(3, 4, 16))),
            "paged": (lambda q: paged_attention(q, cache, *places), (draw(3, 4, 16),))}


def test_forward_mode_and_transforms_are_refused(fake):
    from torch.autograd import forward_ad

    for call, operands in _calls().values():
        for i in range(len(operands)):
            for grad in (False, True):
                with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    ops = [t.clone() for t in operands]
                    ops[i] = forward_ad.make_dual(ops[i], torch.ones_like(ops[i]))
                    with pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
                        call(*ops)
        with pytest.raises(RuntimeError, match="functorch|vmap|data pointer"):
            torch.vmap(lambda t: call(t, *operands[1:]))(operands[0][None].repeat(3, *[1] * operands[0].ndim))


def test_traces_hold_the_operators(fake):
    for name, (call, operands) in _calls().items():
        graph = str(torch.jit.trace(call, operands, check_trace=False).graph)
        assert "^_" in graph, f"{name}: no node for the operator in\n{graph}"


def test_sizes_that_a_launch_does_not_hold():
    """Refused before any launch, the backward's before the forward."""
    meta = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="2\\^26"):
        qk_norm_rotary(meta(1, 1, 1 << 26, 8), meta(1, 1, 1 << 26, 8))
    with pytest.raises(ValueError, match="65535 heads"):
        qk_norm_rotary(meta(1, 65536, 1, 8), meta(1, 1, 1, 8))
    most = (1 << 24) - 8
    shape = lambda B, H, Hk, N, window=0, sinks=0: (ctypes.c_int64 * 18)(  # noqa: E731
        B, H, Hk, N, 8, 0, window, sinks, 0)
    forward = lambda *a: _native.query("tpf_window_forward_workspace_bytes", shape(*a)) >= 0  # noqa: E731
    backward = lambda *a: _native.query("tpf_window_backward_workspace_bytes", shape(*a)) >= 0  # noqa: E731
    assert forward(most // 16, 1, 1, 1) and backward(most // 16, 1, 1, 1)
    assert not forward(most, 1, 1, 1) and not backward(most, 1, 1, 1)
    assert not forward(1, 1, 1, (1 << 30) + 1) and not forward(1, 1 << 20, 1, 1 << 11)
    assert forward(1, 1, 1, 1 << 28) and backward(1, 1, 1, 1 << 20)
    # Sinks take memory for 2048 parts at most, whatever their number is.
    for sinks in (1, 4, 1000, 16383, 16384, 1 << 30):
        size = _native.query("tpf_window_backward_workspace_bytes", shape(1, 4, 1, 16384, 1, sinks))
        assert 0 < size <= (2048 + 128) * 128 * 8 * 8 + 16 * 16384 + 2 * 16384 * 8 * 4 * 16


def test_a_checkpoint_of_other_frequencies_is_told():
    """A block keeps the frequencies that it was made with, and says if they are not the
    checkpoint's."""
    import warnings

    from openfold3_triangle_kernel_amd import SelfAttention

    mine = torch.tensor([0.7, 0.11, 0.03], dtype=torch.float64)
    block, x = SelfAttention(16, 8, 2, frequencies=mine), torch.randn(1, 9, 16)
    want, state = block(x), block.state_dict()
    alike = SelfAttention(16, 8, 2, frequencies=mine)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        alike.load_state_dict(state)
        assert torch.equal(alike(x), want)
        alike.load_state_dict({k: v.bfloat16() for k, v in state.items()})
        alike.load_state_dict({k: v for k, v in state.items() if v.dtype != torch.float64})
        none = [SelfAttention(16, 8, 2, rotary_channels=0) for _ in range(2)]
        none[0].load_state_dict(none[1].state_dict())
    for other in (dict(rotary_channels=6), dict(frequencies=2 * mine), dict(), dict(rotary_channels=0)):
        other = torch.nn.Sequential(SelfAttention(16, 8, 2, **other))
        own = other[0]._frequencies["cpu"].clone()
        with pytest.warns(UserWarning, match="frequencies"):
            other.load_state_dict({"0." + k: v for k, v in state.items()})
        assert torch.equal(other[0]._frequencies["cpu"], own)
        assert torch.equal(other[0].linear_q.weight, block.linear_q.weight)


def test_the_callers_frequencies_are_copied():
    from openfold3_triangle_kernel_amd import SelfAttention

    given = torch.tensor([0.7, 0.11, 0.03], dtype=torch.float64)
    block, x = SelfAttention(16, 8, 2, frequencies=given), torch.randn(1, 9, 16)
    want = block(x)
    given.zero_()
    assert torch.equal(block(x), want)


def test_a_block_is_made_without_memory():
    """Under the meta device, its parameters placed later."""
    from openfold3_triangle_kernel_amd import SelfAttention

    torch.manual_seed(0)
    block, x = SelfAttention(16, 8, 2), torch.randn(1, 9, 16)
    with torch.device("meta"):
        empty = SelfAttention(16, 8, 2)
    assert all(p.is_meta for p in empty.parameters())
    empty.to_empty(device="cpu").load_state_dict(block.state_dict())
    assert torch.equal(empty(x), block(x))


def test_the_last_size_that_a_launch_holds():
    """(2^24 - 8 workgroups of four waves, each with one token or more.)"""
    meta = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="meta")  # noqa: E731
    most = (1 << 26) - 32
    held = PagedCache.of(meta(5, 2, 4, 16), meta(5, 2, 4, 16))
    places = [t.to("meta") for t in _paged()[2:]]
    for T, match in ((most, "GPU"), (most + 1, "2\\^26"), ((1 << 26) - 1, "2\\^26")):
        with pytest.raises(ValueError, match=match):
            qk_norm_rotary(meta(1, 1, T, 8), meta(1, 1, T, 8))
        x = meta(T, 2, 16)
        with pytest.raises(ValueError, match=match):
            append_kv(held, x, x, *places)
        with pytest.raises(ValueError, match=match):
            paged_attention(x, held, *places)
        shape = (ctypes.c_int64 * 25)(1, T, 1, 1, 8, 0, 0, 2, 1, 0, 64)
        size = _native.query("tpf_rotary_backward_workspace_bytes", shape)
        assert size == (768 * 2 * 8 * 4 if T <= most else -1)


def test_the_even_share_of_many_tokens():
    """The join of an even share has a wave a token beside its own workgroups: where a launch
    does not hold them all, the grid is counted from the shapes (without parts here)."""
    cache, _, tables, starts, lengths = _paged(S=2)
    shape = (ctypes.c_int64 * 8)(1, 1, 8, 0, 0, 0, 8, 8)
    for T, even in ((1 << 20, True), ((1 << 26) - 32 - 16384, True), ((1 << 26) - 31 - 16384, False),
                    ((1 << 26) - 36, False)):
        batch = batch_struct(cache.k, tables, starts, lengths, T)
        batch.width, batch.page, batch.pages = 16, 64, 100
        size = _native.query("tpf_paged_attention_workspace_bytes", shape, ctypes.byref(batch))
        assert size == (2 * 1024 * 128 * (8 + 3) * 4 if even else 0)


def test_frequencies_first_used_in_inference_mode_train():
    """A backward keeps the device's copy: it is no inference tensor, whoever makes it."""
    from openfold3_triangle_kernel_amd import SelfAttention

    block = SelfAttention(16, 8, 2)
    with torch.inference_mode():
        copy = block._rotation(torch.device("meta"))
    assert copy is block._rotation(torch.device("meta")) and not copy.is_inference()

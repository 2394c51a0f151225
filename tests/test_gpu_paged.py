"""The paged cache: appended rows against the formulas in 64 bits, places by the tables."""

import pytest
import torch

pytestmark = pytest.mark.gpu

_T = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _batch(dev, news, lengths, page, Hk, D, dtype, behind=0, spare=2, seed=0, width=0):
    """(cache, tables, starts, lengths) of sequences on pages in random order; the cache
    holds random values."""
    from openfold3_triangle_kernel_amd import PagedCache

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).int()
    tables = torch.full((len(need), max(need + [width, 1])), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([sum(news[:s]) for s in range(len(news) + 1)], dtype=torch.int32)
    k, v = (torch.randn(pages, Hk, page, D, generator=g).to(dtype).to(dev) for _ in range(2))
    T = sum(news) + behind
    return PagedCache.of(k, v), tables.to(dev), starts.to(dev), torch.tensor(
        lengths, dtype=torch.int32, device=dev), T, g


APPEND = [
    # new tokens, lengths with them, page, H, Hk, D, half, type, norm, interleaved, rows behind
    ([1], [1], 1, 1, 1, 8, 4, "bf16", True, False, 0),
    ([1, 1, 1], [77, 1, 513], 16, 8, 2, 64, 32, "bf16", True, False, 0),
    ([3, 0, 40, 1], [3, 9, 100, 64], 48, 6, 2, 80, 20, "fp16", False, True, 3),
    ([130, 70], [200, 70], 100, 4, 4, 128, 64, "bf16", True, False, 5),
    ([5] * 70, [20 + s for s in range(70)], 8, 2, 1, 40, 7, "bf16", True, True, 1),
    ([0, 0], [4, 0], 4, 2, 2, 32, 0, "fp16", True, False, 2),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, case):
    from test_gpu_rotary import _check, _frequencies, _reference

    from openfold3_triangle_kernel_amd import append_kv

    news, lengths, page, H, Hk, D, half, t, norm, inter, behind = case
    cache, tables, starts, lens, T, g = _batch(gpu, news, lengths, page, Hk, D, _T[t], behind)
    q, k, v = (torch.randn(T, 2 * h, D, generator=g).to(_T[t]).to(gpu)[:, :h] for h in (H, Hk, Hk))
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(gpu) for _ in range(2)] if norm else [None, None]
    freq = _frequencies(half, gpu) if half else None
    eps = 1e-6 if norm else None
    before = [c.clone() for c in (cache.k, cache.v)]
    out = append_kv(cache, k, v, tables, starts, lens, q, freq, *w, eps, inter)
    live = sum(news)
    assert out.shape == q.shape and out.is_contiguous() and not out[live:].any()
    at = torch.cat([torch.arange(n - m, n) for m, n in zip(news, lengths)] + [torch.zeros(0)]).long()
    seq = torch.cat([torch.full((m,), s) for s, m in enumerate(news)]).long()
    where = tables.cpu()[seq, at // page].long(), at % page
    rows = lambda x: x[:live].transpose(0, 1)[None]  # noqa: E731
    if live:
        _check(rows(out), _reference(rows(q), None, at[None], freq, w[0], eps, inter)[0], "q")
        _check(cache.k[where[0], :, where[1]].transpose(0, 1)[None],
               _reference(rows(k), None, at[None], freq, w[1], eps, inter)[0], "k")
        assert torch.equal(cache.v[where[0], :, where[1]], v[:live])
    for c, b in zip((cache.k, cache.v), before):  # nothing else is written
        c[where[0], :, where[1]] = b[where[0], :, where[1]]
        assert torch.equal(c, b)
    again = append_kv(cache, k, v, tables, starts, lens, None, freq, None, w[1], eps, inter)
    assert again is None


def test_append_without_queries_or_rotation_and_bad_pages(gpu):
    """Values as they are; entries that are no page, and lengths past the table, hold
    nothing."""
    from openfold3_triangle_kernel_amd import append_kv

    cache, tables, starts, lens, T, g = _batch(gpu, [6, 6, 6], [10, 6, 9], 4, 2, 16, torch.bfloat16)
    k, v = (torch.randn(T, 2, 16, generator=g).bfloat16().to(gpu) for _ in range(2))
    tables[0, 2] = cache.pages  # states 8 and 9 of the first sequence
    tables[1, 0] = -5  # states 0 to 3 of the second
    lens[2] = 1000  # the third's tokens lie past its table
    before = [c.clone() for c in (cache.k, cache.v)]
    append_kv(cache, k, v, tables, starts, lens)
    for c, b, x in zip((cache.k, cache.v), before, (k, v)):
        for s, n, m, first in ((0, 10, 6, 0), (1, 6, 6, 6)):
            for i in range(m):
                state = n - m + i
                p = tables[s, state // 4].item()
                if 0 <= p < cache.pages:
                    assert torch.equal(c[p, :, state % 4], x[first + i])
                    b[p, :, state % 4] = x[first + i]
        # The third's length is held to the table's 12 states: its tokens are the last six.
        for i in range(6):
            p = tables[2, (6 + i) // 4].item()
            if 0 <= p < cache.pages:
                b[p, :, (6 + i) % 4] = x[12 + i]
        assert torch.equal(c, b)


def test_append_replays(gpu):
    """A captured append with other tables, lengths and tokens."""
    from openfold3_triangle_kernel_amd import PagedCache, append_kv

    make = lambda seed: _batch(gpu, [1, 1, 1], [9 + seed, 30 - seed, 5 * seed + 1], 8, 2, 32,  # noqa: E731
                               torch.bfloat16, seed=seed, spare=20, width=8)
    cache, tables, starts, lens, T, g = make(0)
    pool = [t[:20].clone() for t in (cache.k, cache.v)]
    cache = PagedCache.of(*pool)
    k, v, q = (torch.randn(T, 2, 32, generator=g).bfloat16().to(gpu) for _ in range(3))
    freq = torch.ones(4, device=gpu)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = append_kv(cache, k, v, tables, starts, lens, q, freq)
    for seed in range(1, 4):
        _, new_tables, _, new_lens, _, g = make(seed)
        tables.copy_(new_tables), lens.copy_(new_lens)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        other = PagedCache.of(*(t.clone() for t in pool))
        want = append_kv(other, k, v, tables, starts, lens, q, freq)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)


ATTEND = [
    # new tokens, lengths with them, page, H, Hk, D, window, sinks, type, rows behind
    ([1], [1], 1, 1, 1, 8, 0, 0, "bf16", 0),
    ([1], [77], 16, 8, 8, 64, 0, 0, "bf16", 0),
    ([1, 1, 1], [700, 3, 1300], 16, 8, 2, 128, 0, 0, "bf16", 2),
    ([1, 1, 1, 1], [2500, 64, 65, 1], 64, 16, 4, 64, 300, 4, "fp16", 0),
    ([1, 0, 1], [5000, 9, 33], 7, 4, 1, 128, 0, 0, "fp16", 1),  # pages that end inside a tile
    ([2, 1, 7], [500, 1, 7], 100, 8, 1, 96, 33, 100, "bf16", 0),
    ([130, 1, 60], [400, 700, 60], 48, 4, 2, 96, 0, 0, "bf16", 5),
    ([300, 5], [1000, 1100], 8, 6, 2, 80, 129, 3, "fp16", 40),
    ([64, 64], [64, 2100], 256, 3, 3, 128, 0, 0, "bf16", 0),
    ([700], [9000], 32, 1, 1, 32, 0, 0, "bf16", 0),
    ([1], [40000], 16, 2, 1, 40, 0, 0, "bf16", 0),  # many parts
    ([1] * 70, [30 + 11 * s for s in range(70)], 8, 2, 1, 64, 50, 1, "bf16", 1),
    ([0, 0, 0], [4, 0, 1], 4, 2, 2, 32, 0, 0, "bf16", 3),
    ([40], [40], 16, 40, 1, 64, 0, 0, "bf16", 0),
]


def _attended(q, cache, tables, news, lengths, window, sinks):
    """The reference of every sequence: (rows, outputs, bounds)."""
    from test_gpu_window_attention import reference, seen

    page, first = cache.page, 0
    for s, (m, n) in enumerate(zip(news, lengths)):
        if m:
            p = tables[s, :-(-n // page)].long()
            k, v = (t[p].transpose(0, 1).reshape(cache.kv_heads, -1, cache.head_dim)[:, :n]
                    for t in (cache.k, cache.v))
            (out,), (err,) = reference(q[first:first + m].transpose(0, 1), k, v,
                                       seen(torch.arange(n - m, n), n, window, sinks),
                                       cache.head_dim ** -0.5)
            yield slice(first, first + m), out.transpose(0, 1), err.transpose(0, 1)
        first += m


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attention(gpu, case):
    from test_gpu_window_attention import check

    from openfold3_triangle_kernel_amd import paged_attention

    news, lengths, page, H, Hk, D, window, sinks, t, behind = case
    cache, tables, starts, lens, T, g = _batch(gpu, news, lengths, page, Hk, D, _T[t], behind)
    q = (1.5 * torch.randn(T, 2 * H, D, generator=g)).to(_T[t]).to(gpu)[:, H:]
    out = paged_attention(q, cache, tables, starts, lens, window or None, sinks)
    assert out.shape == q.shape and out.is_contiguous() and not out[sum(news):].any()
    for rows, want, err in _attended(q, cache, tables, news, lengths, window, sinks):
        check([out[rows]], [want], [err])
    wide = torch.nn.functional.pad(tables, (0, 60), value=-1)  # a longer table splits otherwise
    again = paged_attention(q, cache, wide[:, :-1], starts, lens, window or None, sinks)
    for rows, want, err in _attended(q, cache, tables, news, lengths, window, sinks):
        check([again[rows]], [want], [err])


@pytest.mark.parametrize("group", [1, 3, 5, 40])
@pytest.mark.parametrize("sinks", [0, 1, 64, 129])
def test_attention_spans(gpu, group, sinks):
    """Row tiles whose spans begin and end anywhere in the tiles of states, shared evenly: of
    whole chunks, and of tokens that begin before the first state."""
    from test_gpu_window_attention import check

    from openfold3_triangle_kernel_amd import paged_attention

    news, lengths = [150, 3, 64, 61], [1337, 1200, 64, 1088]
    cache, tables, starts, lens, T, g = _batch(gpu, news, lengths, 16, 1, 32, torch.bfloat16)
    q = torch.randn(T, group, 32, generator=g).bfloat16().to(gpu)
    for window in (1, 2, 63, 64, 65, 127, 1025):
        out = paged_attention(q, cache, tables, starts, lens, window, sinks)
        for rows, want, err in _attended(q, cache, tables, news, lengths, window, sinks):
            check([out[rows]], [want], [err])
    fewer = lens.clone()
    fewer[2] = 20  # 64 new tokens, the last 20 of them states
    out = paged_attention(q, cache, tables, starts, fewer, 65, sinks)
    first = sum(news[:2])
    assert not out[first:first + 44].any() and out[first + 44:first + 64].abs().amax(-1).min() > 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,lengths", [(1, [333, 200]), (60, [333, 200]), (1, [3333, 2000]), (60, [2333, 90])])
def test_attention_never_reads_what_is_not_there(gpu, bad, new, lengths):
    """Places behind a sequence, other pages, pages that the cache does not have and states
    before the window never reach an output, whatever they hold; a later token of the
    chunk never reaches an earlier one."""
    from openfold3_triangle_kernel_amd import PagedCache, paged_attention

    news = [new, new]
    cache, tables, starts, lens, T, g = _batch(gpu, news, lengths, 12, 2, 64, torch.bfloat16)
    q = torch.randn(T, 4, 64, generator=g).bfloat16().to(gpu)
    live = torch.zeros(cache.pages, 12, dtype=torch.bool)
    for s, n in enumerate(lengths):
        for j in range(n):
            live[tables[s, j // 12].item(), j % 12] = True
    dead = ~live.to(gpu)[:, None, :, None]
    clean = PagedCache.of(cache.k.masked_fill(dead, 0), cache.v.masked_fill(dead, 0))
    dirty = PagedCache.of(cache.k.masked_fill(dead, bad), cache.v.masked_fill(dead, bad))
    for window in (None, 40):
        want = paged_attention(q, clean, tables, starts, lens, window)
        got = paged_attention(q, dirty, tables, starts, lens, window)
        assert torch.isfinite(want).all() and torch.equal(got, want)
    # Pages freed behind the window: no entry, or another sequence's page.
    freed = tables.clone()
    for s, n in enumerate(lengths):
        freed[s, :max(0, n - new - 40) // 12] = -1 if s else cache.pages + 7
    assert torch.equal(paged_attention(q, dirty, freed, starts, lens, 40), want)
    # The chunk's last token.
    for t in (dirty.k, dirty.v):
        t[tables[0, (lengths[0] - 1) // 12].item(), :, (lengths[0] - 1) % 12] = bad
    got = paged_attention(q, dirty, tables, starts, lens, None)
    want = paged_attention(q, clean, tables, starts, lens, None)
    rows = torch.ones(T, dtype=torch.bool, device=gpu)
    rows[new - 1] = False
    assert torch.equal(got[rows], want[rows]) and not torch.isfinite(got[new - 1]).all()


def test_attention_without_pages_or_states(gpu):
    """Sequences whose pages the cache does not have, lengths of zero, lengths below the
    new tokens and past the table: zeros, or the states that are there."""
    from openfold3_triangle_kernel_amd import PagedCache, paged_attention

    cache, tables, starts, lens, T, g = _batch(gpu, [3, 3], [40, 50], 8, 1, 32, torch.bfloat16)
    q = torch.randn(T, 2, 32, generator=g).bfloat16().to(gpu)
    want = paged_attention(q, cache, tables, starts, lens)
    none = tables.clone()
    none[0] = 1 << 30
    got = paged_attention(q, cache, none, starts, lens)
    assert not got[:3].any() and torch.equal(got[3:], want[3:])
    for n in (0, -7):
        lens[0] = n
        got = paged_attention(q, cache, tables, starts, lens)
        assert not got[:3].any() and torch.equal(got[3:], want[3:])
    lens[0] = 2  # three tokens, two states: the first token sees none
    got = paged_attention(q, cache, tables, starts, lens)
    assert not got[0].any() and got[1].any() and got[2].any()
    lens[1] = 1 << 30  # held to the table's 56 states: page -1 for the last of them
    assert torch.isfinite(paged_attention(q, cache, tables, starts, lens)).all()
    empty = PagedCache.of(cache.k[:0], cache.v[:0])
    assert not paged_attention(q, empty, tables, starts, lens).any()
    assert not paged_attention(q, cache, tables[:, :0], starts, lens).any()
    assert not paged_attention(q, cache, tables[:0], starts[:1], lens[:0]).any()
    assert paged_attention(q[:0], cache, tables, starts, lens).shape == (0, 2, 32)


def test_starts_that_do_not_ascend(gpu):
    """They get no defined rows, but every access stays in bounds and what follows is right."""
    from openfold3_triangle_kernel_amd import append_kv, paged_attention

    for lengths in ([40, 50, 60], [2000, 50, 60]):
        cache, tables, starts, lens, T, g = _batch(gpu, [2, 2, 2], lengths, 8, 1, 32, torch.bfloat16)
        x = torch.randn(T, 1, 32, generator=g).bfloat16().to(gpu)
        want = paged_attention(x, cache, tables, starts, lens)
        kept = [t.clone() for t in (cache.k, cache.v)]
        for bad in ([0, 5, 2, 6], [3, 2, 1, 0], [-7, 1 << 30, -5, 4], [6, 6, 0, 6]):
            odd = torch.tensor(bad, dtype=torch.int32, device=gpu)
            assert paged_attention(x, cache, tables, odd, lens).shape == x.shape
            append_kv(cache, x, x, tables, odd, lens)
        for t, k in zip((cache.k, cache.v), kept):
            t.copy_(k)
        assert torch.equal(paged_attention(x, cache, tables, starts, lens), want)


@pytest.mark.parametrize("news,length,heads", [
    ([60, 50, 90], 600, 8),      # parts of the states and their join, tiles of many rows
    ([100, 100, 100], 300, 4),   # whole tiles
    ([2] * 70, 520, 8),          # few rows a sequence
    ([7, 30, 1] * 25, 300, 12),  # more sequences than lanes
], ids=str)
def test_starts_that_do_not_ascend_in_tiles_of_many_rows(gpu, news, length, heads):
    """As above outside the even share: tiles and rows that the search finds no sequence for."""
    from openfold3_triangle_kernel_amd import paged_attention

    cache, tables, starts, lens, T, g = _batch(gpu, news, [length] * len(news), 16, 2, 64, torch.bfloat16)
    q = torch.randn(T, heads, 64, generator=g).bfloat16().to(gpu)
    want = paged_attention(q, cache, tables, starts, lens)
    S = len(news)
    cut = starts.clone()
    cut[S // 2 + 1:] = 0
    for bad in (cut, starts.flip(0), starts[torch.randperm(S + 1, generator=g).to(gpu)],
                torch.randint(-T, 2 * T, (S + 1,), generator=g, dtype=torch.int32).to(gpu)):
        assert paged_attention(q, cache, tables, bad.contiguous(), lens).shape == q.shape
    assert torch.equal(paged_attention(q, cache, tables, starts, lens), want)


def test_attention_far_pages(gpu):
    """Pages past 32-bit byte offsets."""
    from openfold3_triangle_kernel_amd import PagedCache, paged_attention

    pages = 540000  # of 16 states of 2 kv heads of 128: 4.4 GB each
    k, v = (torch.zeros(pages, 2, 16, 128, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    g = torch.Generator().manual_seed(4)
    small = [torch.randn(6, 2, 16, 128, generator=g).bfloat16().to(gpu) for _ in range(2)]
    at = torch.tensor([3, pages - 1, 131072, 270001, 524288, 65535], device=gpu)
    k[at], v[at] = small
    starts, lens = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, 5], [90]))
    q = torch.randn(5, 4, 128, generator=g).bfloat16().to(gpu)
    table = torch.arange(6, dtype=torch.int32, device=gpu)[None]
    want = paged_attention(q, PagedCache.of(*small), table, starts, lens)
    assert torch.equal(paged_attention(q, PagedCache.of(k, v), at[None].int(), starts, lens), want)


def test_attention_replays_and_overlaps(gpu):
    """A captured call on other tables, lengths and tokens; calls on two streams."""
    from openfold3_triangle_kernel_amd import paged_attention

    cache, tables, starts, lens, T, g = _batch(gpu, [1, 1, 1], [3000, 700, 1500], 16, 2, 64,
                                               torch.bfloat16, behind=1)
    q = torch.randn(T, 8, 64, generator=g).bfloat16().to(gpu)
    run = lambda: paged_attention(q, cache, tables, starts, lens)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = run()
    for n in ([3000, 700, 1500], [1, 688, 0], [2999, 1, 1024]):
        lens.copy_(torch.tensor(n))
        q.copy_(torch.randn(T, 8, 64, generator=g).bfloat16())
        tables.copy_(tables[:, torch.randperm(tables.shape[1], generator=g).to(gpu)])
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_prompt_then_tokens(gpu):
    """A prompt in chunks and tokens one by one through the cache give the rows of one call
    over all the tokens, to the roundings of both."""
    from test_gpu_window_attention import check, reference, seen

    from openfold3_triangle_kernel_amd import PagedCache, append_kv, paged_attention, qk_norm_rotary

    N, H, Hk, D, window, sinks = 75, 4, 2, 64, 30, 3
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(N, h, D, generator=g).bfloat16().to(gpu) for h in (H, Hk, Hk))
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(gpu)
    freq = 100.0 ** (-torch.arange(16, device=gpu) / 16)
    cache = PagedCache(12, Hk, 8, D)
    table = torch.randperm(12, generator=g).int()[None, :10].to(gpu)
    heads = lambda t: t.transpose(0, 1)  # noqa: E731
    tq, tk = qk_norm_rotary(heads(q)[None], heads(k)[None], None, freq, w, w, 1e-6)
    see = seen(torch.arange(N), N, window, sinks)
    want, err = reference(tq[0], tk[0], heads(v), see, D ** -0.5)
    at = 0
    for new in (33, 1, 30, 1, 1, 1, 8):
        rows = slice(at, at + new)
        at += new
        starts, lens = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, new], [at]))
        turned = append_kv(cache, k[rows], v[rows], table, starts, lens, q[rows], freq, w, w, 1e-6)
        assert torch.equal(turned, heads(tq[0])[rows])
        out = paged_attention(turned, cache, table, starts, lens, window, sinks)
        check([heads(out)], [want[0][:, rows]], [err[0][:, rows]])


def test_append_to_nothing(gpu):
    """A cache without pages, tables without entries, no sequences: queries are turned all the
    same where they have a sequence, and nothing is written."""
    from openfold3_triangle_kernel_amd import PagedCache, append_kv

    cache, tables, starts, lens, T, g = _batch(gpu, [3, 3], [40, 50], 8, 1, 32, torch.bfloat16)
    q, k = (torch.randn(T, 1, 32, generator=g).bfloat16().to(gpu) for _ in range(2))
    freq = torch.tensor([1.0, 0.1], dtype=torch.float64, device=gpu)
    before = [t.clone() for t in (cache.k, cache.v)]
    want = append_kv(PagedCache.of(*(t.clone() for t in before)), k, k, tables, starts, lens, q, freq)
    empty = PagedCache.of(cache.k[:0], cache.v[:0])
    assert torch.equal(append_kv(empty, k, k, tables, starts, lens, q, freq), want)
    lens.clamp_(max=0)  # (what a table without entries holds)
    short = append_kv(cache, k, k, tables[:, :0], starts, lens, q, freq)
    assert torch.equal(short, append_kv(cache, k, k, tables, starts, lens, q, freq))
    assert not append_kv(cache, k, k, tables[:0], starts[:1], lens[:0], q, freq).any()
    assert append_kv(cache, k[:0], k[:0], tables, starts, lens, q[:0]).shape == (0, 1, 32)
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])

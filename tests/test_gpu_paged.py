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

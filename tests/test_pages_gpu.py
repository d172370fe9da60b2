"""Forking and compacting pages against the definitions, one row after the other: every value equal."""

from __future__ import annotations

import pytest
import torch

from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu


def _cache(rows, N, page, width, planes, longest, per_row, seed=0, prefix=0):
    """Rows of random lengths (some empty), ids drawn without regard to each other, a common prefix."""
    g = torch.Generator().manual_seed(seed)
    pages = torch.randn(planes, N, page, width, generator=g).to(torch.bfloat16)
    table = torch.randint(0, N, (rows, per_row), generator=g, dtype=torch.int32)
    if prefix and rows:
        table[:, :prefix] = table[0, :prefix].clone()
    lens = torch.randint(0, longest + 1, (rows,), generator=g, dtype=torch.int32)
    return pages, table, lens


def _fork(be, pages, table, lens, parent, add, keep=None, strides=None):
    want = orc.fork(pages, table, lens, parent.tolist(), add.tolist(), [] if keep is None else keep.tolist())
    p = pages.cuda() if strides is None else strides(pages)
    t, n = table.cuda(), lens.cuda()
    got = be.fork_pages(p, t, n, parent.cuda(), add.cuda(), None if keep is None else keep.cuda())
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b), (a.cpu(), b)
    assert torch.equal(p.cpu(), want[3])
    assert torch.equal(t.cpu(), table) and torch.equal(n.cpu(), lens)
    return got


def _compact(be, pages, table, lens, keep=None):
    want = orc.compact(pages, table, lens, [] if keep is None else keep.tolist())
    p = pages.cuda()
    got = be.compact_pages(p, table.cuda(), lens.cuda(), None if keep is None else keep.cuda())
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    live = int(got[2])
    # Places past the live ones keep what they held.
    assert torch.equal(p.cpu(), want[3]) and torch.equal(p.cpu()[:, live:], pages[:, live:])


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("page,width,planes", [(16, 128, 2), (32, 640, 4), (64, 8, 1), (1024, 24, 2)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_fork_random(hip_backend, page, width, planes, seed):
    rows = (1, 7, 40)[seed]
    g = torch.Generator().manual_seed(100 + seed)
    pages, table, lens = _cache(rows, 12 * rows + 9, page, width, planes, 5 * page, 8, seed, prefix=seed)
    out = rows + seed
    parent = torch.randint(-1, rows, (out,), generator=g, dtype=torch.int32)
    add = torch.randint(0, 2 * page, (out,), generator=g, dtype=torch.int32)
    _fork(hip_backend, pages, table, lens, parent, add)
    _fork(hip_backend, pages, table, lens, parent, add, keep=torch.randint(-2, 12 * rows, (11,), generator=g, dtype=torch.int32))


def test_fork_copies_only_the_tokens_of_a_shared_written_page(hip_backend):
    pages, table, _ = _cache(2, 20, 16, 64, 2, 0, 4)
    table[0, :2], table[1, :2] = _ints(5, 6), _ints(7, 8)
    lens = _ints(21, 32)
    # Row 0 twice (a copy each), row 1 twice (its last page is full: shared, no copy), row 0 without new tokens.
    t, n, status = _fork(hip_backend, pages, table, lens, _ints(0, 0, 1, 1, 0), _ints(1, 1, 1, 1, 0))
    assert t[:, 1].tolist() == [0, 1, 8, 8, 6] and t[2:4, 2].tolist() == [2, 3]
    # A row alone writes in place.
    t, n, status = _fork(hip_backend, pages, table, lens, _ints(0, 1), _ints(11, 0))
    assert t[0, :2].tolist() == [5, 6]
    # ... unless `keep` holds the page.
    t, n, status = _fork(hip_backend, pages, table, lens, _ints(0, 1), _ints(1, 0), keep=_ints(6))
    assert t[0, :2].tolist() == [5, 0]


def test_fork_defaults(hip_backend):
    pages, table, lens = _cache(5, 60, 16, 64, 2, 40, 4)
    want = orc.fork(pages, table, lens, range(5), [3] * 5)
    p = pages.cuda()
    got = hip_backend.fork_pages(p, table.cuda(), lens.cuda(), add=3)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and torch.equal(p.cpu(), want[3])
    got = hip_backend.fork_pages(p, table.cuda(), lens.cuda())
    want = orc.fork(want[3], table, lens, range(5), [0] * 5)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and torch.equal(p.cpu(), want[3])


def test_fork_when_pages_run_out(hip_backend):
    pages, table, _ = _cache(3, 6, 16, 64, 2, 0, 4)
    table[0, :2], table[1, :1], table[2, :1] = _ints(0, 1), _ints(1), _ints(2)
    lens = _ints(20, 10, 16)
    got = _fork(hip_backend, pages, table, lens, _ints(0, 1, 2, 2), _ints(1, 1, 17, 40))
    assert int(got[2][0]) == 0 and int(got[2][1]) > 0
    # ... and when a row is full.
    got = _fork(hip_backend, pages, table, lens, _ints(2, 2, 1), _ints(60, 0x7FFFFFFF, 1))
    assert int(got[2][1]) > 0


def test_fork_bad_entries(hip_backend):
    pages, table, lens = _cache(6, 40, 16, 64, 2, 60, 4)
    table[0, 0], table[1, 1], table[2, 0], table[3, 3] = -1, 40, 1 << 30, -(1 << 31)
    lens[4], lens[5] = 1 << 30, -5
    _fork(hip_backend, pages, table, lens, _ints(0, 1, 2, 3, 4, 5, 6, -9, 1 << 30), _ints(1, 1, 1, -1, 1, 1, 1, 1, 1),
          keep=_ints(-1, 40, 3, 1 << 30))


def test_fork_from_and_to_nothing(hip_backend):
    pages, table, lens = _cache(3, 40, 16, 64, 2, 60, 4)
    _fork(hip_backend, pages, table, lens, _ints(), _ints())  # every sequence ends
    empty = torch.full((0, 4), -1, dtype=torch.int32), _ints()
    _fork(hip_backend, pages, *empty, _ints(-1, -1, 0), _ints(1, 0, 64))
    _fork(hip_backend, pages, *empty, _ints(), _ints())


def test_fork_strided_pages(hip_backend):
    """Planes inside pages, and padded pages."""
    pages, table, lens = _cache(9, 60, 16, 64, 4, 60, 5, seed=4)
    parent, add = torch.arange(9, dtype=torch.int32) // 2, torch.ones(9, dtype=torch.int32)
    _fork(hip_backend, pages, table, lens, parent, add, strides=lambda p: p.transpose(0, 1).contiguous().cuda().transpose(0, 1))

    def padded(p):
        wide = torch.zeros(4, 60, 1032, dtype=torch.bfloat16, device="cuda")
        view = wide[:, :, :1024].unflatten(2, (16, 64))
        view.copy_(p)
        return view

    _fork(hip_backend, pages, table, lens, parent, add, strides=padded)


@pytest.mark.parametrize("N", [1, 63, 1024, 1025, 5000, 300000])
def test_fork_cache_sizes(hip_backend, N):
    pages, table, lens = _cache(12, N, 16, 8, 1, 200, 16, seed=N)
    _fork(hip_backend, pages, table, lens, torch.arange(12, dtype=torch.int32) // 3, torch.full((12,), 5, dtype=torch.int32))
    _compact(hip_backend, pages, table, lens)


def test_many_rows(hip_backend):
    pages, table, lens = _cache(2500, 9000, 16, 8, 1, 40, 3, seed=6)
    g = torch.Generator().manual_seed(1)
    parent = torch.randint(-1, 2500, (3001,), generator=g, dtype=torch.int32)
    _fork(hip_backend, pages, table, lens, parent, torch.randint(0, 9, (3001,), generator=g, dtype=torch.int32))
    _compact(hip_backend, pages, table, lens)


@pytest.mark.parametrize("page,width,planes", [(16, 128, 2), (32, 640, 4), (64, 8, 1), (1024, 24, 2)])
@pytest.mark.parametrize("rows", [1, 5, 33])
def test_compact_random(hip_backend, page, width, planes, rows):
    pages, table, lens = _cache(rows, 10 * rows + 3, page, width, planes, 4 * page, 6, rows, prefix=2)
    _compact(hip_backend, pages, table, lens)
    _compact(hip_backend, pages, table, lens, keep=_ints(0, 10 * rows + 2, 10 * rows + 3, -1, 4, 4))


def test_compact_full_empty_and_tidy_caches(hip_backend):
    pages, table, _ = _cache(4, 16, 16, 64, 2, 0, 4)
    table[:] = torch.randperm(16, generator=torch.Generator().manual_seed(2)).view(4, 4)
    _compact(hip_backend, pages, table, _ints(64, 64, 64, 64))
    _compact(hip_backend, pages, table, _ints(0, 0, 0, 0))
    table[:] = torch.arange(16).view(4, 4)
    _compact(hip_backend, pages, table, _ints(64, 50, 0, 0))
    _compact(hip_backend, pages, table[:0].contiguous(), _ints())


def test_compact_bad_entries(hip_backend):
    pages, table, lens = _cache(6, 40, 16, 64, 2, 60, 4)
    table[0, 0], table[1, 1], table[2, 0] = -1, 40, 1 << 30
    lens[4], lens[5] = 1 << 30, -5
    _compact(hip_backend, pages, table, lens)


def test_pool_past_32_bit_offsets(hip_backend):
    """Copies between pages that lie 5 GiB apart."""
    N, page, width = 10500, 1024, 256
    pages = torch.zeros(1, N, page, width, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(8)
    content = torch.randn(3, page, width, generator=g).to(torch.bfloat16)
    ids = [N - 1, 4100, 8200]
    pages[0, ids] = content.cuda()
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    lens = torch.tensor([3 * page - 1], dtype=torch.int32, device="cuda")
    t, n, status = hip_backend.fork_pages(pages, table, lens, torch.zeros(2, dtype=torch.int32, device="cuda"), 1)
    assert t.tolist() == [[N - 1, 4100, 0], [N - 1, 4100, 1]] and status.tolist() == [N - 5, 0]
    assert torch.equal(pages[0, 0, : page - 1].cpu(), content[2, : page - 1]) and not pages[0, 0, page - 1].any()
    t, where, live = hip_backend.compact_pages(pages, table, lens)
    assert t.tolist() == [[2, 0, 1]] and int(live) == 3
    assert torch.equal(pages[0, :3].cpu(), content[[1, 2, 0]])


def test_captured(hip_backend):
    pages, table, lens = _cache(8, 80, 16, 64, 2, 60, 5, seed=11)
    p, t, n = pages.cuda(), table.cuda(), lens.cuda()
    parent, add = torch.arange(8, dtype=torch.int32, device="cuda") // 2, torch.ones(8, dtype=torch.int32, device="cuda")
    hip_backend.fork_pages(p.clone(), t, n, parent, add)
    hip_backend.compact_pages(p.clone(), t, n)
    torch.cuda.synchronize()
    graph, tidy = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = hip_backend.fork_pages(p, t, n, parent, add)
    p2 = pages.cuda()
    with torch.cuda.graph(tidy):
        got2 = hip_backend.compact_pages(p2, t, n)
    for step in range(4):
        g = torch.Generator().manual_seed(step)
        parent.copy_(torch.randint(-1, 8, (8,), generator=g, dtype=torch.int32))
        p.copy_(pages)
        p2.copy_(pages)
        graph.replay()
        tidy.replay()
        torch.cuda.synchronize()
        want = orc.fork(pages, table, lens, parent.tolist(), [1] * 8)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and torch.equal(p.cpu(), want[3])
        want = orc.compact(pages, table, lens)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got2, want)) and torch.equal(p2.cpu(), want[3])


@pytest.mark.parametrize("N,rows,per_row", [(700, 100, 600), (700, 50, 600), (5000, 70, 600), (40000, 300, 350), (270000, 3, 40)])
def test_many_entries_in_few_pages_and_few_in_many(hip_backend, N, rows, per_row):
    """Both sides of where the whole chip counts holders: entries against pages."""
    page = 16
    g = torch.Generator().manual_seed(N + rows)
    pages, table, lens = _cache(rows, N, page, 8, 2, per_row * page - 200, per_row, seed=rows, prefix=3)
    lens[::7] = 0
    if N < 1000:  # leave pages free: rows of ten ids between them
        table = table % 10 + 3
        table[:, 2] = 690
    parent = torch.randint(-1, rows, (rows,), generator=g, dtype=torch.int32)
    add = torch.randint(0, 40, (rows,), generator=g, dtype=torch.int32)
    keep = torch.tensor([N - 1, 5, -1, N], dtype=torch.int32)
    _fork(hip_backend, pages, table, lens, parent, add, keep)
    _compact(hip_backend, pages, table, lens, keep)


def test_compact_pages_of_one_word_and_of_all_words(hip_backend):
    """Held pages at the words' ends: 31, 32, 33, the last, and none in between."""
    for N in (31, 32, 33, 64, 1000, 33000):
        pages = torch.arange(2 * N, dtype=torch.float32).view(2, N, 1, 1).expand(2, N, 16, 8).to(torch.bfloat16).contiguous()
        ids = sorted({i for i in (0, 30, 31, 32, 33, 63, N - 2, N - 1) if 0 <= i < N})
        table = torch.tensor([ids[::-1]], dtype=torch.int32)
        _compact(hip_backend, pages, table, _ints(16 * len(ids)))
        _fork(hip_backend, pages, table, _ints(16 * len(ids) - 5), _ints(0, 0), _ints(1, 1))

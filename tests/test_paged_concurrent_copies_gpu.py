"""Forks that copy pages and compactions that move them, called at once: the copies' list and the pages
themselves, on streams of their own, from threads, in graphs replayed side by side."""

from __future__ import annotations

import threading

import pytest
import torch

from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu

PAGE, WIDTH, PER_ROW = 16, 512, 8


def _inputs(seed, rows, num):
    g = torch.Generator().manual_seed(seed)
    pages = torch.randn(4, num, PAGE, WIDTH, generator=g).to(torch.bfloat16)
    lens = torch.randint(1, PER_ROW * PAGE - 20, (rows,), generator=g, dtype=torch.int32)
    table = orc.page_table(lens.tolist(), PAGE, PER_ROW, num, seed)
    return g, pages, table, lens


class _Fork:
    """Every row continued about twice and written: a copy for each child of a partly filled page."""

    def __init__(self, be, seed):
        rows = 24 + seed
        g, self.pages, table, lens = _inputs(seed, rows, 400 + 16 * seed)
        parent = torch.randint(0, rows, (2 * rows,), generator=g, dtype=torch.int32)
        self.want = orc.fork(self.pages, table, lens, parent.tolist(), [1] * len(parent))
        assert int(self.want[2][1]) == 0 and not torch.equal(self.want[3], self.pages)
        table, lens, parent = table.cuda(), lens.cuda(), parent.cuda()
        self.op = lambda pool: be.fork_pages(pool, table, lens, parent, 1)
        self.saved, self.pool = self.pages.cuda(), self.pages.cuda()

    def __call__(self):
        self.pool.copy_(self.saved)
        return self.op(self.pool) + (self.pool,)


class _Compact(_Fork):
    """Live pages all over the cache: most of them move."""

    def __init__(self, be, seed):
        _, self.pages, table, lens = _inputs(seed, 24 + seed, 400 + 16 * seed)
        self.want = orc.compact(self.pages, table, lens)
        assert not torch.equal(self.want[3], self.pages)
        table, lens = table.cuda(), lens.cuda()
        self.op = lambda pool: be.compact_pages(pool, table, lens)
        self.saved, self.pool = self.pages.cuda(), self.pages.cuda()


def _fine(call, got):
    return all(torch.equal(a.cpu(), b) for a, b in zip(got, call.want, strict=True))


@pytest.mark.parametrize("pair", [(_Fork, _Fork), (_Compact, _Compact), (_Fork, _Compact)])
def test_two_streams_at_once(hip_backend, pair):
    calls = [make(hip_backend, s) for s, make in enumerate(pair)]
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                *out, pool = c()
                got[i].append((*out, pool.clone()))  # the pool is restored by the next call
    torch.cuda.synchronize()
    for c, all_got in zip(calls, got):
        assert all(_fine(c, x) for x in all_got)


@pytest.mark.parametrize("make", [_Fork, _Compact])
def test_threads_call_at_once(hip_backend, make):
    calls = [make(hip_backend, s) for s in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = calls[i]()
                torch.cuda.current_stream().synchronize()
                if not _fine(calls[i], got):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("pair", [(_Fork, _Fork), (_Compact, _Compact), (_Fork, _Compact)])
def test_two_graphs_replayed_side_by_side(hip_backend, pair):
    calls = [make(hip_backend, s) for s, make in enumerate(pair)]
    for c in calls:
        c()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(4):
        for c in calls:
            c()  # eager work between the replays
        torch.cuda.synchronize()
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(_fine(c, out) for c, out in zip(calls, outs))

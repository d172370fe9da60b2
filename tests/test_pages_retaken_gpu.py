"""A fork that ran out of pages, taken again from the old table: what it left whole."""

from __future__ import annotations

import pytest
import torch

from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu

PAGE = 16


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _start():
    """Three rows of 20, 20 and 10 tokens in six pages, one of them free, and each row's tokens."""
    pages = torch.randn(2, 6, PAGE, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    table = torch.full((3, 6), -1, dtype=torch.int32)
    table[0, :2], table[1, :2], table[2, :1] = _ints(0, 1), _ints(2, 3), _ints(4)
    lens = _ints(20, 20, 10)
    return pages, table, lens, [_tokens(pages, table[i], n) for i, n in enumerate(lens.tolist())]


def _tokens(pages, row, n):
    ids = row[: -(-n // PAGE)].long().cpu()
    assert bool((ids >= 0).all())
    return pages.cpu()[:, ids].flatten(1, 2)[:, :n]


def _run_out(be, pool, table, lens, keep):
    """Both children of row 0 ask for more than the cache holds."""
    _, _, status = be.fork_pages(pool, table, lens, _ints(0, 0).cuda(), 60, keep)
    assert int(status[1]) > 0


def test_rows_that_the_call_continued_are_whole(hip_backend):
    pages, table, lens, tokens = _start()
    pool, table, lens = pages.cuda(), table.cuda(), lens.cuda()
    _run_out(hip_backend, pool, table, lens, None)
    assert torch.equal(_tokens(pool, table[0], 20), tokens[0])
    t, n, status = hip_backend.fork_pages(pool, table, lens, _ints(0, 0).cuda(), 1)
    assert status.tolist() == [2, 0] and n.tolist() == [20, 20]
    assert all(torch.equal(_tokens(pool, t[i], 20), tokens[0]) for i in (0, 1))


def test_kept_rows_are_whole_and_may_be_continued_instead(hip_backend):
    pages, table, lens, tokens = _start()
    pool, table, lens = pages.cuda(), table.cuda(), lens.cuda()
    _run_out(hip_backend, pool, table, lens, _ints(0, 1, 2, 3, 4).cuda())
    parent = [1, 2, 1]
    want = orc.fork(pool.cpu(), table.cpu(), lens.cpu(), parent, [1] * 3)
    t, n, status = hip_backend.fork_pages(pool, table, lens, _ints(*parent).cuda(), 1)
    assert torch.equal(t.cpu(), want[0]) and torch.equal(status.cpu(), want[2]) and int(status[1]) == 0
    for i, p in enumerate(parent):
        assert torch.equal(_tokens(pool, t[i], int(n[i])), tokens[p])

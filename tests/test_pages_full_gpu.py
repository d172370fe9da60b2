"""Compaction of caches whose every page is held, where the whole chip counts holders."""

from __future__ import annotations

import pytest
import torch

from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("num", [700, 1023, 1024, 1025, 2048, 2500])
@pytest.mark.parametrize("free", [0, 1])
def test_every_page_held(hip_backend, num, free):
    """Whole runs of pages for each of the plan's 1,024 threads, and a part of one; with one page free, too."""
    page, per_row, rows = 16, 700, 70  # more entries than one work-group takes
    g = torch.Generator().manual_seed(num)
    pages = torch.randn(2, num, page, 8, generator=g).to(torch.bfloat16)
    table = torch.randint(0, num, (rows, per_row), generator=g, dtype=torch.int32)
    table.view(-1)[:num] = torch.randperm(num, generator=g)
    if free:
        table[table == num // 3] = 0
    lens = torch.full((rows,), per_row * page, dtype=torch.int32)
    want = orc.compact(pages, table, lens)
    assert int(want[2]) == num - free
    pool = pages.cuda()
    for _ in range(3):
        pool.copy_(pages)
        got = hip_backend.compact_pages(pool, table.cuda(), lens.cuda())
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and torch.equal(pool.cpu(), want[3])

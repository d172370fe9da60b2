"""The choice of pages where little is left to choose."""

from __future__ import annotations

import pytest
import torch

from tests import drafts_oracle as drafts
from tests.test_sparse_attention_gpu import _attend, _case, _choice, _stale

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [5, 300, 3000, 9000])
def test_the_last_page_alone(hip_backend, pages):
    """Through every form of the choice; bounds are not read: NaN ones give the same."""
    q, k, v, table, lens = _case([1, 37, 16 * 5, 0, 70], 8, 2, 64, 16, per_row=pages)
    limit = _stale(k)
    ref = _choice(hip_backend, q, limit, table, lens, 1, 16)
    _attend(hip_backend, q, k, v, limit, table, lens, 1)
    got = hip_backend.select_pages(q.cuda(), torch.full_like(limit, float("nan")).cuda(), table.cuda(), lens.cuda(), 1, 16)
    assert torch.equal(got[0].cpu(), ref[0]) and torch.equal(got[1].cpu(), ref[1])

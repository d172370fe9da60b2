"""The choice of pages where little is left to choose."""

from __future__ import annotations

import pytest
import torch

from tests.test_sparse_attention_gpu import _attend, _bounds, _case, _choice, _stale

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


@pytest.mark.parametrize("H,G", [(4, 2), (16, 2)])
@pytest.mark.parametrize("zero", [False, True])
def test_pages_with_a_channel_without_a_number_come_last(hip_backend, H, G, zero):
    """Whatever their other channels say: the bounds of such a channel are low = inf, high = -inf, and its term -inf,
    or, with a query of zero there, no number."""
    page, count = 16, 4
    q, k, v, table, lens = _case([160], H, G, 64, page)
    k[table[0, 3].long(), :, :, 2] = 1e4  # would be the best
    q[..., 2] = 1.0
    k[table[0, 3].long(), :, 0, 5] = float("nan")  # kv head 0
    k[table[0, 6].long(), 0, 0, 5] = float("nan")  # one token of them: left out
    k[table[0, 6].long(), 1:, :, 2] = 9e3
    if zero:
        q[..., 5] = 0.0
    limit = hip_backend.key_bounds(k.cuda(), _stale(k).cuda(), table.cuda(), lens.cuda())
    at = table[0, 3].long()
    assert limit[at, 0, :, 5].tolist() == [float("inf"), float("-inf")]
    ref = _choice(hip_backend, q, limit.cpu(), table, lens, count, page)
    first, second = ref[0][0, 0].tolist(), ref[0][0, 1].tolist()
    assert int(at) not in first and int(at) in second and int(table[0, 6]) in first
    # Taken where nothing else is left, the earliest such pages first.
    everything, _ = hip_backend.select_pages(q.cuda(), limit, table.cuda(), lens.cuda(), 9, page)
    assert int(at) not in everything[0, 0].tolist()
    k[table[0, 7].long(), :, 0, 8] = float("nan")
    limit = hip_backend.key_bounds(k.cuda(), limit, table.cuda(), lens.cuda())
    everything, _ = hip_backend.select_pages(q.cuda(), limit, table.cuda(), lens.cuda(), 9, page)
    assert int(at) in everything[0, 0].tolist() and int(table[0, 7]) not in everything[0, 0].tolist()


@pytest.mark.parametrize("page", [16, 128])
def test_bounds_of_lengths_and_firsts_outside_the_row(hip_backend, page):
    """A length far beyond the row ends at the row's end, one below zero is none, and neither is anything left behind
    a ``first`` beyond the length."""
    _, k, _, table, _ = _case([4 * page] * 4, 2, 2, 64, page, per_row=4)
    lens = torch.tensor([1 << 30, -7, 2**31 - 1, 3 * page + 1], dtype=torch.int32)
    _bounds(hip_backend, k, table, lens)
    _bounds(hip_backend, k, table, lens, torch.tensor([1 << 30, 0, 3 * page, -(1 << 31)], dtype=torch.int32))
    _bounds(hip_backend, k, table, lens, torch.tensor([4 * page, 5, 2 * page - 1, 3 * page + 1], dtype=torch.int32))

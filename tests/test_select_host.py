"""What the choice of pages needs, without a GPU."""

from __future__ import annotations

import pytest

from breezetoken_amd import _lib


@pytest.mark.parametrize("batch,kv_heads,pages", [(1, 1, 2), (3, 2, 40), (128, 8, 9000)])
def test_scores_take_room_only_where_there_is_something_to_choose(batch, kv_heads, pages):
    """One page is the last one, and a row of as many pages as are kept keeps them."""
    size, sparse = _lib.lib().bt_select_workspace_bytes, _lib.lib().bt_sparse_workspace_bytes
    assert size(batch, kv_heads, pages, 1) == 0 and size(batch, kv_heads, pages, pages) == 0
    if pages > 2:
        assert size(batch, kv_heads, pages, 2) >= batch * kv_heads * pages * 8
    # The choice, its lengths and what the attention over one page needs, whatever the width of the table.
    assert sparse(batch, 8 * kv_heads, kv_heads, 128, pages, 16, 1) == sparse(batch, 8 * kv_heads, kv_heads, 128, 2, 16, 1)

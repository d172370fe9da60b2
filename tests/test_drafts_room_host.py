"""What the operators over drafts and selected pages need and refuse, without a GPU."""

from __future__ import annotations

import pytest

from breezetoken_amd import _lib
from tests.test_drafts_host import ACCEPT, SELECT
from tests.test_paged_host import A, PREP


@pytest.mark.parametrize("batch,kv_heads,pages", [(1, 1, 2), (3, 2, 40), (128, 8, 9000)])
def test_scores_take_room_only_where_there_is_something_to_choose(batch, kv_heads, pages):
    """One page is the last one, and a row of as many pages as are kept keeps them."""
    size, sparse = _lib.lib().bt_select_workspace_bytes, _lib.lib().bt_sparse_workspace_bytes
    assert size(batch, kv_heads, pages, 1) == 0 and size(batch, kv_heads, pages, pages) == 0
    if pages > 2:
        assert size(batch, kv_heads, pages, 2) >= batch * kv_heads * pages * 8
    # The choice, its lengths and what the attention over one page needs, whatever the width of the table.
    assert sparse(batch, 8 * kv_heads, kv_heads, 128, pages, 16, 1) == sparse(batch, 8 * kv_heads, kv_heads, 128, 2, 16, 1)


@pytest.mark.parametrize("name", ["table", "lens", "parents", "tokens", "first", "best", "lens_out", "path", "following"])
def test_accept_refuses_unaligned_integers(name):
    assert _lib.lib().bt_accept_drafts(*{**ACCEPT, name: ACCEPT[name] + 2}.values()) == -22


def test_select_refuses_unaligned_lengths():
    assert _lib.lib().bt_select_pages(*{**SELECT, "chosen_lens": SELECT["chosen_lens"] + 2}.values()) == -22


def test_prep_of_drafts_refuses_unaligned_angles():
    at = list(PREP).index("rows")
    assert _lib.lib().bt_attn_prep_drafts(*list(PREP.values())[:at], A + 2, *list(PREP.values())[at:]) == -22

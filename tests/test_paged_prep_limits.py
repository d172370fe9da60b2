"""Rows of the projection that 32-bit numbers of their values do not reach are refused; nothing is launched."""

from __future__ import annotations

import pytest

from breezetoken_amd import _lib
from tests.test_paged_host import PREP


@pytest.mark.parametrize("heads,kv_heads,gated,dim", [(1 << 21, 1, 1, 512), (1 << 22, 1, 0, 512), (1, 1 << 21, 0, 512),
                                                      (1 << 23, 1, 1, 128), (1 << 24, 1, 0, 128), (1 << 24, 1, 1, 64)])
def test_rows_past_32_bits_are_refused(heads, kv_heads, gated, dim):
    row = heads * dim * (1 + gated) + 2 * kv_heads * dim
    assert row > 2**31 - 1
    # Whatever else is wrong is refused as -22 before: the strides and the cache here are fine.
    call = {**PREP, "stride": row, "tokens": 1, "heads": heads, "kv_heads": kv_heads, "dim": dim, "gated": gated,
            "sp": 16 * kv_heads * dim, "st": kv_heads * dim, "sh": dim, "rope": 64}
    assert _lib.lib().bt_attn_prep_paged(*call.values()) == -95

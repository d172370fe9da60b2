"""Attention of drafted tokens at the ends of what is served: the largest batch and head dimension together."""

from __future__ import annotations

import pytest
import torch

from tests.test_tree_attention_gpu import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("longest", [40, 5000])
def test_largest_batch_of_the_largest_heads(hip_backend, longest):
    """4,096 sequences' running sums beside two tiles of K and V in LDS: parts of one sequence and, with a longer row,
    more places than one."""
    lens = [b % 3 for b in range(4096)]
    lens[1234] = longest
    _check(hip_backend, *_case(lens, 1, 1, 1, 256, 16, per_row=400, parents=torch.full((4096, 1), -1, dtype=torch.int32)))

"""Attention of drafted tokens whose sequence is cut into parts: what the join has to keep of every part."""

from __future__ import annotations

import pytest
import torch

from tests.test_tree_attention_gpu import _case, _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("batch,length,token", [(24, 2400, 51), (5, 700, 30), (1, 9000, 100), (1, 9000, 8990), (3, 120, 20)])
def test_a_cached_value_without_a_number_counts_whatever_its_parts_weight(hip_backend, batch, length, token, what):
    """The other half of the keys lies 2^1400 above the one that has it: its channel is infinite or NaN all the same."""
    H, G, D, page = 8, 2, 64, 16
    q, k, v, table, lens, parents = _case([length] * batch, 4, H, G, D, page, per_row=640, parents=torch.tensor([[-1, 0, 0, -1]] * batch, dtype=torch.int32))
    q[..., 0] = 8.0
    b, low = batch // 2, token < length // 2
    for t in range(length + 4):
        above = t >= length // 2 if low else t < length // 2
        k[table[:, t // page].long(), t % page, :, 0] = 1000.0 if above else 0.0
    v[table[b, token // page], token % page, 0, 7] = float(what)
    got = _run(hip_backend, q, k, v, table, lens, parents).cpu()
    assert not got[b, :, : H // G, 7].isfinite().any()
    got[b, :, : H // G, 7] = 0
    assert got.isfinite().all()


@pytest.mark.parametrize("batch,short,longest", [(64, 20, 9000), (64, 300, 9000), (130, 40, 5000), (31, 40, 12000), (3, 10, 30000), (2, 10, 60000)])
@pytest.mark.parametrize("D", [64, 256])
def test_one_long_sequence_among_short_ones(hip_backend, batch, short, longest, D):
    """Most of the parts are one sequence's."""
    lens = [short] * batch
    lens[batch // 3] = longest
    _check(hip_backend, *_case(lens, 2, 2, 1, D, 64))

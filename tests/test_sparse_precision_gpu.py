"""Results of sparse attention in bf16: rounded once, from 24 bits, for any number of heads a kv head."""

from __future__ import annotations

import pytest
import torch

from tests import drafts_oracle as drafts
from tests.test_sparse_attention_gpu import _case, _stale

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (32, 8, 128), (5, 1, 64), (16, 2, 256), (16, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,count", [([1, 37, 301, 0, 130], 6), ([3000, 17, 1604], 90)])
def test_bf16_results_are_the_f32_results_rounded(hip_backend, H, G, D, q_dtype, lens, count):
    """Whole sequences and parts; the f32 results are held to 64 bits elsewhere."""
    q, k, v, table, n = _case(lens, H, G, D, 16, q_dtype=q_dtype)
    limit = drafts.bounds(k, _stale(k), table, lens)
    dev = [t.cuda() for t in (q, k, v, limit, table, n)]
    full = hip_backend.attention_sparse(*dev, count, D**-0.5)
    assert torch.equal(hip_backend.attention_sparse(*dev, count, D**-0.5, out_dtype=torch.bfloat16), full.to(torch.bfloat16))

"""A prompt's tokens behind a prefix that several sequences share: written into pages, then attended
with a table row for each token."""

from __future__ import annotations

import pytest
import torch

from breezetoken_amd import PagedKVCache
from breezetoken_amd.backend import rope_tables
from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix,chunks", [(37, (5, 20, 1)), (64, (33, 2)), (1, (16,))])
def test_prompt_chunks_behind_a_shared_prefix(hip_backend, prefix, chunks):
    be, H, G, D, page = hip_backend, 8, 2, 128, 16
    g = torch.Generator().manual_seed(prefix)
    cache = PagedKVCache(40, page, G, D, "cuda")
    k, v = cache.layer(0)
    cos, sin = rope_tables(200, 64, 1.0e4, "cuda")
    table, lens = cache.empty_table(1, 160)
    table, lens, status = be.fork_pages(cache.pages, table, lens, add=prefix)

    def write(rows, pos):
        qkv = torch.randn(len(pos), (H + 2 * G) * D, generator=g).cuda()
        q, _ = be.attn_prep_paged(qkv, None, None, 0.0, cos, sin, pos, 64, k, v, table, H, G, D, rows=rows, gated=False)
        return q

    write(torch.zeros(prefix, dtype=torch.int32, device="cuda"), torch.arange(prefix, dtype=torch.int32, device="cuda"))
    lens = lens + prefix
    # Every prompt continues row 0 and gets room for its own tokens.
    sizes = torch.tensor(chunks, dtype=torch.int32, device="cuda")
    table, lens, status = be.fork_pages(cache.pages, table, lens, torch.zeros_like(sizes), sizes)
    assert int(status[1]) == 0
    rows = torch.repeat_interleave(torch.arange(len(chunks), device="cuda"), sizes.long()).to(torch.int32)
    pos = torch.cat([prefix + torch.arange(n) for n in chunks]).to(torch.int32).cuda()
    q = write(rows, pos)
    got = be.attention_paged(q, k, v, table[rows.long()], pos + 1, D**-0.5)
    args = [t.cpu() for t in (q, k, v, table[rows.long()], pos + 1)]
    want = orc.attention(*args, D**-0.5)
    tol = orc.attention_tolerance(args[0], args[1], args[2], D**-0.5, prefix + max(chunks), want, False)
    assert bool(((got.double().cpu() - want).abs() <= tol).all())

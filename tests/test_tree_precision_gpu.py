"""Attention of drafted tokens in 24 bits: inputs whose products are exact, so that what is left is the rounding of
queries, probabilities and results, tight enough to tell three bf16 terms of a value from two."""

from __future__ import annotations

import math

import pytest
import torch

from tests import drafts_oracle as drafts
from tests import paged_oracle as orc
from tests.test_tree_attention_gpu import _case

pytestmark = pytest.mark.gpu

F32 = orc.F32
LOG2E = 1.0 / math.log(2.0)


def two_keys(length: int, drafts_: int, reach: tuple[float, float], q_dtype=torch.float32, seed: int = 0):
    """(q, k, v, table, lens, parents): of ``length`` cached tokens the first and the last count, with scores of 0 and
    ``reach`` (in log2) and values in channels of their own; the others lie 2^-400 and more below them.

    A score is one product with a power of two, exact apart from the query's own rounding."""
    g = torch.Generator().manual_seed(seed)
    H, G, D, page = 8, 2, 64, 16
    pages = -(-(length + drafts_) // page)
    k = torch.zeros(pages, page, G, D)
    v = torch.zeros(pages, page, G, D)
    flat_k, flat_v = k.view(-1, G, D), v.view(-1, G, D)
    flat_k[1 : length - 1, :, 1] = -1.0  # channel 1 of the queries: 512
    flat_k[length - 1, :, 0] = 1.0
    flat_k[length:, :, 1] = -1.0
    flat_v[0, :, 0], flat_v[length - 1, :, 1] = 1.0, 1.0
    flat_v[1 : length - 1, :, 2:] = 1.0
    low, high = reach
    q = torch.zeros(1, drafts_, H, D)
    q[..., 0] = (low + (high - low) * torch.rand(1, drafts_, H, generator=g)) / LOG2E
    q[..., 1] = 512.0
    table = torch.arange(pages, dtype=torch.int32)[None]
    parents = torch.full((1, drafts_), -1, dtype=torch.int32)
    return q.to(q_dtype), k.bfloat16(), v.bfloat16(), table, torch.tensor([length], dtype=torch.int32), parents


def expected(q: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The two channels that are not zero, in 64 bits: the keys' shares."""
    x = q[..., 0].double()
    return 1 / (1 + torch.exp(x)), 1 / (1 + torch.exp(-x))


def tolerance(q: torch.Tensor, joined: bool) -> torch.Tensor:
    """Relative, for either channel.

    The scale in log2, the query's product with it, the sum of its three terms and the difference from the reference
    round to half a step each, relative to the score: a share moves by ln 2 times that at most.  To it come, in half steps: two
    exponentials (2 each, a step), the probability's three terms' sum and its residual (2), the sum of the
    probabilities (2), the division (1) and the product with it (1), and the result's own (1).  Joined, lse and its
    difference from the largest (a logarithm 2, the sum's rounding 1 and the difference's 1, relative to a few units
    of log2, 5 at most here: 20 ln 2), two more exponentials (4), products and sums (4) and a division (1)."""
    x = (q[..., 0].double() * LOG2E).abs()
    return (4 * math.log(2) * x + 11 + (20 * math.log(2) + 9 if joined else 0)) * F32


REACHES = [(-1.0, 1.0), (-20.0, -12.0), (12.0, 20.0)]


@pytest.mark.parametrize("reach", REACHES)
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("length,drafts_", [(2, 64), (31, 64), (100, 28)])
def test_f32_results(hip_backend, length, drafts_, q_dtype, reach):
    """Shares of two keys, by the one work-group that has all of them."""
    q, *rest = two_keys(length, drafts_, reach, q_dtype)
    got = hip_backend.attention_tree(q.cuda(), *(t.cuda() for t in rest), 1.0).double().cpu()
    for channel, ref in enumerate(expected(q)):
        off = (got[..., channel] - ref).abs() / ref
        assert float((off - tolerance(q, False)).max()) <= 0, (channel, float(off.max()) / F32)
    assert not got[..., 2:].any()


@pytest.mark.parametrize("length,drafts_", [(600, 64), (3000, 64), (9000, 8)])
def test_f32_results_of_joined_parts(hip_backend, length, drafts_):
    """The two keys lie in the first and the last of several parts."""
    q, *rest = two_keys(length, drafts_, (-1.0, 1.0))
    got = hip_backend.attention_tree(q.cuda(), *(t.cuda() for t in rest), 1.0).double().cpu()
    for channel, ref in enumerate(expected(q)):
        off = (got[..., channel] - ref).abs() / ref
        assert float((off - tolerance(q, True)).max()) <= 0, (channel, float(off.max()) / F32)


def _half_step(x: torch.Tensor) -> torch.Tensor:
    """Half of the distance between bf16 values at x, which is not zero."""
    return torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent - 9)


def near_borders(seed: int):
    """``two_keys`` whose second share, a probability that is not 1, lies beside the middle of two bf16 values, one and
    a half tolerances off it."""
    q, *rest = two_keys(60, 64, (-1.0, 1.0), seed=seed)
    share = expected(q)[1]
    middle = share.bfloat16().double() + _half_step(share)
    g = torch.Generator().manual_seed(seed)
    side = 2.0 * torch.randint(0, 2, share.shape, generator=g) - 1
    share = middle * (1 + 1.5 * side * tolerance(q, False))
    q[..., 0] = torch.log(share / (1 - share)).float()
    return q, *rest


@pytest.mark.parametrize("seed", range(4))
def test_bf16_results(hip_backend, seed):
    """Rounded once, from 24 bits: further off than half a step by no more than f32 results are."""
    q, *rest = near_borders(seed)
    got = hip_backend.attention_tree(q.cuda(), *(t.cuda() for t in rest), 1.0, out_dtype=torch.bfloat16).double().cpu()
    ref = expected(q)[1]
    off = (got[..., 1] - ref).abs()
    assert float((off - _half_step(ref) - tolerance(q, False) * ref).max()) <= 0


@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (32, 8, 128), (12, 12, 64), (16, 2, 128)])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 37, 301, 0, 130], [1800, 700, 2500]])
def test_bf16_results_are_the_f32_results_rounded(hip_backend, H, G, D, q_dtype, lens):
    dev = [t.cuda() for t in _case(lens, 16, H, G, D, 32, q_dtype=q_dtype)]
    full = hip_backend.attention_tree(*dev, D**-0.5)
    assert torch.equal(hip_backend.attention_tree(*dev, D**-0.5, out_dtype=torch.bfloat16), full.to(torch.bfloat16))


@pytest.mark.parametrize("factor", [1.0, 40.0])
def test_as_near_as_f32_sums(hip_backend, factor):
    """Ordinary inputs, and scores forty times as large: at most four times the error of the formula in f32 with its
    sums in another order (two bf16 terms of the queries: twelve times and more, of the probabilities nine times, or,
    where the scores' own rounding is forty times as large, one term a hundred times)."""
    q, k, v, table, lens, parents = _case([70, 5], 16, 8, 2, 128, 16)
    q = q * factor
    ref = drafts.attention_tree(q, k, v, table, lens, parents, 128**-0.5)
    got = hip_backend.attention_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), parents.cuda(), 128**-0.5)
    assert float((got.double().cpu() - ref).abs().max()) <= 4 * float((f32_form(q, k, v, table, lens, parents) - ref).abs().max())


def f32_form(q, k, v, table, lens, parents) -> torch.Tensor:
    """Every draft by itself, sums in 32 bits."""
    B, T, H, D = q.shape
    page, G = k.shape[1:3]
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        for i, line in enumerate(drafts.ancestors(parents[b].tolist())):
            if line is None:
                continue
            slots = torch.tensor(list(range(n)) + [n + j for j in sorted(line)])
            ids, at = table[b, slots // page].long(), slots % page
            for h in range(H):
                x = (k[ids, at, h // (H // G)].float() * q[b, i, h]).sum(dim=1) * D**-0.5
                e = torch.exp(x - x.max())
                out[b, i, h] = ((e / e.sum())[:, None] * v[ids, at, h // (H // G)].float()).sum(dim=0).double()
    return out

"""Beam selection against a sort of every candidate in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu


def _check(be, logits, scores, beams=None):
    count = logits.shape[1] if beams is None else beams
    want = orc.beams(logits, scores, count)
    got = be.beam_select(logits.cuda(), scores.cuda(), beams)
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])
    value, ref = got[0].cpu().double(), want[0]
    ref = torch.where(ref < torch.finfo(torch.float32).min, -math.inf, ref)  # past f32's range: -inf
    fine = ref.isfinite()
    assert torch.equal(value[~fine], ref[~fine])
    # The result's own rounding, and 2^-22 for the log of the sum.
    assert bool(((value - ref).abs()[fine] <= ref.abs()[fine] * orc.F32 + 2.0**-22).all())
    return got


def _case(B, W, V, dtype=torch.float32, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, W, V, generator=g) * spread).to(dtype), -10 * torch.rand(B, W, generator=g)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 4097, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabularies(hip_backend, V, dtype):
    _check(hip_backend, *_case(2, 3, V, dtype, V), 3)


@pytest.mark.parametrize("W,beams", [(1, 1), (1, 5), (4, 4), (5, 1), (8, 16), (3, 64), (64, 64), (64, 3), (17, 13)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widths(hip_backend, W, beams, dtype):
    _check(hip_backend, *_case(3, W, 901, dtype, W * 100 + beams), beams)


@pytest.mark.parametrize("V,dtype", [(248320, torch.float32), (248320, torch.bfloat16), (100003, torch.float32)])
def test_large_vocabularies(hip_backend, V, dtype):
    _check(hip_backend, *_case(1, 2, V, dtype, 5), 4)


def test_many_searches(hip_backend):
    _check(hip_backend, *_case(150, 2, 300, seed=2), 2)


@pytest.mark.parametrize("beams", [1, 4, 40])
@pytest.mark.parametrize("V", [50, 5000])
def test_ties_go_to_the_lower_place(hip_backend, beams, V):
    logits = torch.zeros(2, 3, V)
    _check(hip_backend, logits, torch.zeros(2, 3), beams)
    logits[:, :, ::3] = 1.0
    _check(hip_backend, logits, torch.zeros(2, 3), beams)
    _check(hip_backend, torch.randint(-2, 3, (2, 3, V), generator=torch.Generator().manual_seed(1)).float(),
           torch.tensor([[0.0, -1.0, 0.0], [-3.0, -3.0, -3.0]]), beams)
    logits = torch.zeros(1, 1, V)
    logits[0, 0, ::2] = -0.0  # equal to +0
    _check(hip_backend, logits, torch.zeros(1, 1), beams)


@pytest.mark.parametrize("order", ["up", "down"])
def test_sorted_logits(hip_backend, order):
    """Every value a new best one, and none after the first."""
    x = torch.linspace(-8, 8, 20000)
    x = x if order == "up" else x.flip(0)
    _check(hip_backend, x.repeat(2, 2, 1), torch.tensor([[0.0, -0.3], [-5.0, 0.1]]), 2)
    _check(hip_backend, x.repeat(1, 2, 1), torch.tensor([[0.0, -0.3]]), 64)


def test_barred_tokens_and_ended_beams(hip_backend):
    logits, scores = _case(2, 4, 3000, seed=3)
    logits[:, :, torch.randperm(3000, generator=torch.Generator().manual_seed(0))[:2500]] = -math.inf
    logits[0, 1] = -math.inf
    logits[0, 1, 7] = 0.0  # an ended beam keeps its score
    got = _check(hip_backend, logits, scores, 6)
    scores[0, 1] = 5.0
    got = _check(hip_backend, logits, scores, 6)
    assert int(got[1][0, 0]) == 1 and int(got[2][0, 0]) == 7 and float(got[0][0, 0]) == 5.0


def test_infinite_and_nan_logits(hip_backend):
    logits, scores = _case(4, 3, 100, seed=4)
    logits[0] = -math.inf  # nothing left: candidates of -inf, lowest places
    logits[1, 0] = float("nan")
    logits[1, 1, ::2] = float("nan")
    logits[2, 0, 5] = math.inf
    logits[2, 1] = math.inf
    logits[3, 0] = torch.finfo(torch.float32).min
    want_first = math.log(1.0)
    want = []
    got = [t.cpu() for t in hip_backend.beam_select(logits.cuda(), scores.cuda(), 5)]
    ref = orc.beams(torch.cat((logits[:2], logits[3:])), torch.cat((scores[:2], scores[3:])), 5)
    for i, b in enumerate((0, 1, 3)):
        assert torch.equal(got[1][b].long() - 3 * b, ref[1][i] - 3 * i) and torch.equal(got[2][b].long(), ref[2][i])
    # +inf: one token takes all of beam 0, a hundred share beam 1.  With the most beams both are among the chosen.
    got = [t.cpu() for t in hip_backend.beam_select(logits.cuda(), scores.cuda(), 64)]
    value = {(0, 5): float(scores[2, 0]) - want_first, (1, 0): float(scores[2, 1]) - math.log(100)}
    for v, p, t in zip(got[0][2].tolist(), got[1][2].tolist(), got[2][2].tolist()):
        if (p - 6, t) in value:
            want.append(abs(v - value[(p - 6, t)]))
    assert len(want) == 2 and max(want) <= 2.0**-20
    assert not any(t.isnan().any() for t in got[:1])


def test_infinite_scores(hip_backend):
    """The first step of a search: one live beam, the others at -inf."""
    logits, scores = _case(2, 4, 500, seed=6)
    scores[:, 1:] = -math.inf
    got = _check(hip_backend, logits, scores, 4)
    assert got[1][:, :].cpu().tolist() == [[0] * 4, [4] * 4]
    _check(hip_backend, logits[:, :, :2], scores, 8)  # all candidates


def test_extreme_logits(hip_backend):
    g = torch.Generator().manual_seed(12)
    logits = torch.randn(2, 2, 700, generator=g) * 1e4
    _check(hip_backend, logits, torch.zeros(2, 2), 5)
    logits = torch.randn(2, 2, 700, generator=g) * 1e-30
    _check(hip_backend, logits, torch.tensor([[0.0, -1.0], [-2.0, 0.0]]), 5)
    logits = torch.full((1, 1, 700), torch.finfo(torch.float32).min)
    logits[0, 0, 3] = torch.finfo(torch.float32).max
    _check(hip_backend, logits, torch.zeros(1, 1), 2)


def test_strided_logits(hip_backend):
    logits, scores = _case(3, 4, 1001, seed=7)
    want = [t.cpu() for t in hip_backend.beam_select(logits.cuda(), scores.cuda())]
    wide = torch.zeros(4, 3, 1010, device="cuda")
    wide[:, :, 3:1004] = logits.transpose(0, 1).cuda()
    views = (wide[:, :, 3:1004].transpose(0, 1), logits.cuda().transpose(1, 2).contiguous().transpose(1, 2))
    for x in views:
        got = hip_backend.beam_select(x, scores.cuda())
        assert all(torch.equal(a, b.cpu()) for a, b in zip(want, got))
    one = logits[:1, :1].cuda().expand(2, 3, 1001)  # one set of logits for every beam
    _check(hip_backend, one.cpu(), scores[:2, :3])
    for lead in (1, 2, 3, 5):  # rows that begin at any alignment
        x = torch.randn(2, 2, 300, generator=torch.Generator().manual_seed(lead)).to(torch.bfloat16)
        wide = torch.zeros(2, 2, 311, dtype=torch.bfloat16, device="cuda")
        wide[:, :, lead : lead + 300] = x.cuda()
        a = hip_backend.beam_select(wide[:, :, lead : lead + 300], scores[:2, :2].cuda())
        b = hip_backend.beam_select(x.cuda(), scores[:2, :2].cuda())
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_repeated_and_captured(hip_backend):
    logits, scores = (t.cuda() for t in _case(2, 4, 30000, seed=8))
    first = hip_backend.beam_select(logits, scores)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip_backend.beam_select(logits, scores)
    for step in range(4):
        logits.copy_(torch.randn(2, 4, 30000, generator=torch.Generator().manual_seed(step)) * 2)
        graph.replay()
        eager = hip_backend.beam_select(logits, scores)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        assert all(torch.equal(a.cpu().long(), b) for a, b in zip(out[1:], orc.beams(logits.cpu(), scores.cpu(), 4)[1:]))
    assert not torch.equal(first[2], out[2])


def test_no_searches(hip_backend):
    got = hip_backend.beam_select(torch.zeros(0, 3, 9, device="cuda"), torch.zeros(0, 3, device="cuda"), 2)
    assert [tuple(t.shape) for t in got] == [(0, 2)] * 3


def _check_values(be, logits, scores, beams):
    """The same where candidates of different beams are equal but for the order of their sums' terms.  A row's
    log-sum is off by e = 2^-22 at most, and beams are ordered by these values: the i-th of them is within e of
    the i-th exact one, and the exact value of the candidate chosen for it within e of that."""
    got = be.beam_select(logits.cuda(), scores.cuda(), beams)
    value = torch.log_softmax(logits.double(), -1) + scores.double()[..., None]
    value = torch.where(value.isnan(), -math.inf, value)  # a row barred whole
    B, W, V = value.shape
    want = value.view(B, -1).sort(descending=True).values[:, :beams]
    at = (got[1].cpu().long() % W) * V + got[2].cpu().long()
    mine = value.view(B, -1).gather(1, at)
    assert all(len(set(x.tolist())) == beams for x in at)
    fine = want.isfinite()
    assert torch.equal(mine.isfinite(), fine) and torch.equal(got[0].cpu().isfinite(), fine)
    assert bool(((mine - want).abs()[fine] <= 2 * 2.0**-22).all())
    off = (got[0].cpu().double() - mine).abs()
    assert bool((off[fine] <= mine.abs()[fine] * orc.F32 + 2.0**-22).all())


@pytest.mark.parametrize("W,beams,V", [(64, 64, 300), (40, 64, 70), (20, 20, 3000), (33, 1, 500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_equal_candidates(hip_backend, W, beams, V, dtype):
    """Logits of few values and equal scores: more candidates reach any bound than lists hold."""
    g = torch.Generator().manual_seed(W)
    logits = torch.randint(0, 2, (2, W, V), generator=g).to(dtype)
    logits[1] = 0.5
    _check(hip_backend, logits[1:], torch.zeros(1, W), beams)
    _check_values(hip_backend, logits, torch.zeros(2, W), beams)
    logits[0, : W // 2] = -math.inf  # barred whole: they come last
    logits[0, W // 2 :, 3:] = -math.inf
    _check_values(hip_backend, logits, torch.zeros(2, W), beams)


@pytest.mark.parametrize("W,beams", [(32, 32), (64, 64), (48, 10), (2, 64)])
def test_wide_searches(hip_backend, W, beams):
    _check(hip_backend, *_case(2, W, 20000, torch.bfloat16, seed=W), beams)
    _check(hip_backend, *_case(2, W, 9001, seed=W), beams)

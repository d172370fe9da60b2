"""Beam selection's log-sums where the mass lies far below the largest logit."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# A logit's exponential is taken relative to the largest of sixteen.  The exponent's rounding moves the sixteen's
# sum by 2^-24 at most: terms of 2^-a of the largest are off by 2^-24 a ln 2, and weigh 15 x 2^-a together.  The
# missing part of log2(e) moves it by a third of that, v_exp by 2^-23, three f32 additions by 2^-24 each, the
# factor's rounding by 2^-24; all further sums are in 64 bits.  7.3 x 2^-24 together.
LOG_SUM = 2.0**-21


def _flat_rows(top, low, V, dtype):
    """Rows of one logit `top` and V - 1 of `low`; the log-sum less `top`, in 64 bits."""
    top, low = top.to(dtype), low.to(dtype)
    x = low.cuda()[:, None].expand(len(top), V).clone()
    x[:, V // 3] = top.cuda()
    return x, torch.log1p((V - 1) * torch.exp(low.double() - top.double()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [32000, 248320])
@pytest.mark.parametrize("batch", [1, 17])  # 17: so many rows that one work-group, and one reference, takes a whole one
@pytest.mark.parametrize("near,far", [(6.0, 9.0), (9.0, 11.0), (11.1, 12.4)])
def test_a_peak_above_equal_logits(hip_backend, dtype, V, batch, near, far):
    g = torch.Generator().manual_seed(int(far * 10))
    W = 64
    top = torch.rand(W, generator=g) * 40 - 20
    low = top - near - (far - near) * torch.rand(W, generator=g)
    top[0], low[0] = 7.30921, -3.6139622
    x, less = _flat_rows(top, low, V, dtype)
    # Scores that leave of each row's best candidate little but its sum's error, a step apart: the order is theirs.
    scores = (less + torch.arange(W) * 2.0**-19).float()
    exact = scores.double() - less
    logits = x.expand(batch, W, V)
    got, parent, token = (t.cpu() for t in hip_backend.beam_select(logits, scores.cuda().expand(batch, W).contiguous(), W))
    assert bool((token == V // 3).all())
    rows = parent.long() % W
    assert float((got.double() - exact[rows]).abs().max()) <= LOG_SUM
    # Exact values are at least 2^-19 - 2^-20 apart (the scores' own rounding), both sums off by LOG_SUM at most.
    assert bool((rows == torch.arange(W - 1, -1, -1)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch", [1, 17])
def test_shapes_of_mass(hip_backend, dtype, batch):
    """Steps of equal logits, spread ones, and sixteens that hold one large logit each."""
    V, W = 50000, 6
    g = torch.Generator().manual_seed(5)
    x = torch.empty(W, V)
    x[0] = torch.linspace(-14, 0, V)
    x[1] = -torch.arange(V).float().remainder(16)
    x[2] = -11.37
    x[2, ::16] = 3.21
    x[3] = torch.randn(V, generator=g) * 5
    x[4] = torch.randn(V, generator=g).abs() * -3 - 80
    x[5] = -4000.3
    x[5, 7] = -3990.1
    x = x.to(dtype)
    less = torch.logsumexp(x.double(), 1) - x.double().max(1).values
    scores = less.float()
    logits = x.cuda().expand(batch, W, V)
    for w in range(W):  # one row live at a time
        s = torch.full((batch, W), -math.inf)
        s[:, w] = scores[w]
        got, parent, _ = (t.cpu() for t in hip_backend.beam_select(logits, s.cuda(), 1))
        assert bool((parent[:, 0] == torch.arange(batch) * W + w).all())
        assert float((got.double() - (scores[w].double() - less[w])).abs().max()) <= LOG_SUM


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch", [1, 17])
@pytest.mark.parametrize("order", [0, 1, 2])
def test_stretches_of_different_size(hip_backend, dtype, batch, order):
    """Rows of stretches that no common reference suits: near 0, near the largest, thousands below it, barred,
    not a number; a stretch's logits within three of one another.  Largest logits up to 4,096 and past it."""
    V, W, piece = 70001, 64, 1777
    g = torch.Generator().manual_seed(order)
    levels = torch.tensor([0.0, 11.0, -300.0, 4.0, -5000.0, -math.inf, math.nan, 7.5, -90.0])
    x = torch.randn(W, V, generator=g).clamp(-3, 3)
    for at in range(0, V, piece):
        x[:, at : at + piece] += levels[torch.randint(0, len(levels), (W, 1), generator=g)]
    x += torch.tensor([0.0, 4080.0, -3900.0, 30000.0, -6000.0, 1.0e6])[torch.arange(W) % 6][:, None]
    if order == 1:
        x = x.sort(dim=1).values  # NaN last
    elif order == 2:
        x = x.nan_to_num(-math.inf, None, -math.inf).sort(dim=1, descending=True).values
    x = x.to(dtype)
    clean = torch.where(x.isnan(), -math.inf, x.double())
    top = clean.max(1).values
    less = torch.log(torch.exp(clean - top[:, None]).sum(1))
    scores = less.float() - 60 * torch.arange(W)  # every row's best candidates before the next row's
    exact = scores.double() - less
    got, parent, token = (t.cpu() for t in hip_backend.beam_select(x.cuda().expand(batch, W, V),
                                                                   scores.cuda().expand(batch, W).contiguous(), 64))
    first = clean.argmax(1)  # the lowest of equal ones
    for b in range(batch):
        assert int(parent[b, 0]) == b * W and int(token[b, 0]) == int(first[0])
        assert abs(float(got[b, 0]) - float(exact[0])) <= LOG_SUM
        # The order inside the row, and values: 64 candidates of row 0.
        best = torch.sort(clean[0], descending=True, stable=True)
        assert torch.equal(token[b].long(), best.indices[:64]) and bool((parent[b] == b * W).all())
        want = best.values[:64] - top[0] + exact[0]
        assert float((got[b].double() - want).abs().max()) <= LOG_SUM + float(want.abs().max()) * 2.0**-24
    for w in range(1, W, 5):
        s = torch.full((batch, W), -math.inf)
        s[:, w] = less[w].float()
        got, parent, token = (t.cpu() for t in hip_backend.beam_select(x.cuda().expand(batch, W, V), s.cuda(), 1))
        assert bool((token == first[w]).all()) and bool((parent[:, 0] == torch.arange(batch) * W + w).all())
        assert float((got.double() - (less[w].float().double() - less[w])).abs().max()) <= LOG_SUM

"""YaRN's tables, every pair of them, against the method's definition."""

from __future__ import annotations

import math

import pytest
import torch

from breezetoken_amd.backend import rope_tables_scaled


def _rates(rope_dim: int, theta: float, factor: float, trained: float) -> tuple[list[float], list[float]]:
    """Each pair's angle a position, and how often it turns over the trained context unscaled.

    Pair i turns trained theta^(-2i/rope_dim) / 2 pi times, so n times where i is
    rope_dim log(trained / (2 pi n)) / (2 log theta)."""
    rates, turns = [], []
    at = [rope_dim * math.log(trained / (2 * math.pi * n)) / (2 * math.log(theta)) for n in (32, 1)]
    first, last = math.floor(at[0]), math.ceil(at[1])
    for i in range(rope_dim // 2):
        rate = theta ** (-2 * i / rope_dim)
        turns.append(trained * rate / (2 * math.pi))
        ramp = min(1.0, max(0.0, (i - first) / (last - first)))
        rates.append(rate * (1 - ramp) + rate / factor * ramp)
    return rates, turns


@pytest.mark.parametrize("trained", [4, 150, 4096, 32768, 65536, 131072, 1 << 20])
@pytest.mark.parametrize("rope_dim,theta", [(128, 1.0e4), (64, 1.0e4), (64, 1.0e7), (10, 500.0)])
@pytest.mark.parametrize("factor", [4.0, 32.0])
def test_yarn_tables(rope_dim, theta, factor, trained):
    cos, sin = rope_tables_scaled(40, rope_dim, theta, "yarn", factor, trained, "cpu")
    rates, turns = _rates(rope_dim, theta, factor, trained)
    scale = 0.1 * math.log(factor) + 1.0
    pos = torch.arange(40, dtype=torch.float64)[:, None]
    angle = pos * torch.tensor(rates, dtype=torch.float64)
    half = rope_dim // 2
    for got, want in ((cos, angle.cos() * scale), (sin, angle.sin() * scale)):
        assert float((got[:, :half].double() - want).abs().max()) <= scale * 2.0**-24 + 1e-12
        assert torch.equal(got[:, :half], got[:, half:])
    # The words of the definition: rates read back from the tables, position 1.
    back = torch.atan2(sin[1, :half].double(), cos[1, :half].double())
    for i, n in enumerate(turns):
        plain = theta ** (-2 * i / rope_dim)
        if n >= 32:
            assert abs(float(back[i]) - plain) <= 2.0**-22
        elif n <= 1:
            assert abs(float(back[i]) - plain / factor) <= 2.0**-22
        else:
            assert plain / factor - 2.0**-22 <= float(back[i]) <= plain + 2.0**-22


@pytest.mark.parametrize("trained", [None, 0, -1, math.inf, math.nan])
def test_trained_lengths_that_are_none(trained):
    with pytest.raises(ValueError, match="trained context"):
        rope_tables_scaled(16, 64, 1.0e4, "yarn", 8.0, trained, "cpu")

"""What the paged decode's f32 arithmetic may be off, row by row, tight enough to tell how many
bf16 terms queries and probabilities are held in; checked here on the CPU, by the arithmetic
restated, and used by the GPU tests."""

from __future__ import annotations

import math

import pytest
import torch

F32 = 2.0**-24  # half a step, relative


def rows(lens, H, G, D, page, per_row, q_dtype=torch.float32, seed=0):
    """Inputs of a call, K and V of every sequence in pages of its own."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    N = sum(used) + 2
    k, v = (torch.randn(N, page, G, D, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(len(lens), H, D, generator=g).to(q_dtype)
    ids = torch.randperm(N, generator=g).to(torch.int32)
    table = torch.full((len(lens), per_row), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at : at + n]
        at += n
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32)


def keys_of(k, v, table, lens, b):
    page, G, D = k.shape[1:]
    n = int(lens[b])
    ids = table[b, : -(-n // page)].long()
    return k[ids].reshape(-1, G, D)[:n], v[ids].reshape(-1, G, D)[:n]


def result_and_tolerance(q, k, v, table, lens, scale: float):
    """(B, H, D) in 64 bits, and what f32 arithmetic may move each value.

    Roundings are of random sign, at most half a step of what they round: 3^-1/2 of that in the
    mean square.  A score s = scale * q . k takes D of them at partial sums that grow to
    S = |q * k| * scale (a random walk) or |s|, half of that in the mean square, one of each scaled
    query value, and further ones at |s| (the scale's own), at its distance to the largest (the
    exponent) and at 1 (the exponential); they move probability p by that much of itself, and the
    result by p (v - o).  The sum over the keys takes a rounding per key at partial sums that grow
    to |p v| and |o|, and the end a few at |o|.  Six times the root of the mean square, for the
    largest of 10^5 values."""
    B, H, D = q.shape
    G = k.shape[2]
    out, tol = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        if int(lens[b]) < 1:
            continue
        keys, values = keys_of(k, v, table, lens, b)
        for h in range(H):
            kk, vv = keys[:, h // (H // G)].double(), values[:, h // (H // G)].double()
            prod = kk * q[b, h].double() * scale
            s, S = prod.sum(1), prod.norm(dim=1)
            p = torch.softmax(s, 0)
            o = p @ vv
            size = torch.maximum(S, s.abs())
            off = F32 * (math.sqrt((D + 2) / 6) * size + s.abs() + (s.max() - s) / math.log(2) + 2)
            moved = ((p * off)[:, None] * (vv - o)).norm(dim=0)
            partial = (p[:, None] * vv).norm(dim=0) + o.abs()
            out[b, h] = o
            tol[b, h] = 6 * (moved + F32 * math.sqrt(len(s) / 6) * partial + F32 * o.abs())
    return out, tol


def in_terms(q, k, v, table, lens, scale: float, terms: int) -> torch.Tensor:
    """The kernel's arithmetic in f32: scaled queries and probabilities as sums of bf16 terms."""

    def split(x):
        parts = []
        for _ in range(terms):
            parts.append(x.to(torch.bfloat16).float())
            x = x - parts[-1]
        return parts

    B, H, D = q.shape
    G = k.shape[2]
    out = torch.zeros(B, H, D)
    for b in range(B):
        keys, values = keys_of(k, v, table, lens, b)
        for h in range(H):
            kk, vv = keys[:, h // (H // G)].float(), values[:, h // (H // G)].float()
            x = sum(kk @ t for t in split(q[b, h].float() * torch.tensor(scale * math.log2(math.e))))
            p = torch.exp2(x - x.max())
            out[b, h] = sum(t @ vv for t in split(p)) / p.sum()
    return out


def rounds_to(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor) -> torch.Tensor:
    """Where a bf16 result is what some value within ``tol`` of ``want`` rounds to."""
    low, high = ((want + sign * tol).to(torch.float32).to(torch.bfloat16).double() for sign in (-1, 1))
    return (got.double() >= low) & (got.double() <= high)


CASES = [((2, 5, 17, 40, 130), 8, 2, 256), ((3, 33, 64, 200), 7, 1, 128), ((4, 9, 100), 15, 5, 64), ((6, 31, 90), 16, 2, 128)]


@pytest.mark.parametrize("lens,H,G,D", CASES)
@pytest.mark.parametrize("spread", [1.0, 6.0])
def test_three_terms_pass_and_two_do_not(lens, H, G, D, spread):
    q, k, v, table, n = rows(lens, H, G, D, 16, 16)
    q = q * spread
    want, tol = result_and_tolerance(q, k, v, table, n, D**-0.5)
    worst = [float(((in_terms(q, k, v, table, n, D**-0.5, t).double() - want).abs() / tol).max()) for t in (3, 2)]
    assert worst[0] <= 0.5 and worst[1] >= 1.3, worst


def test_bf16_results_tell_the_terms_too():
    lens = [40 + 7 * (b % 11) for b in range(20)]
    q, k, v, table, n = rows(lens, 16, 4, 128, 16, 8, torch.bfloat16)
    want, tol = result_and_tolerance(q, k, v, table, n, 128**-0.5)
    fine = [rounds_to(in_terms(q, k, v, table, n, 128**-0.5, t).to(torch.bfloat16), want, tol) for t in (3, 2)]
    assert bool(fine[0].all()) and int((~fine[1]).sum()) >= 2

"""The paged decode's precision: within what f32 arithmetic may be off, which two bf16 terms are not."""

from __future__ import annotations

import pytest
import torch

from tests.test_paged_precision import result_and_tolerance, rounds_to, rows

pytestmark = pytest.mark.gpu


def _run(be, args, dtype):
    scale = args[0].shape[-1] ** -0.5
    want, tol = result_and_tolerance(*args, scale)
    return be.attention_paged(*(t.cuda() for t in args), scale, out_dtype=dtype).cpu(), want, tol


# Rows of up to 512 tokens (whole sequences) and of 2,048 (runs).
@pytest.mark.parametrize("per_row", [16, 128])
@pytest.mark.parametrize("H,G,D,q_dtype", [(16, 4, 128, torch.bfloat16), (16, 4, 128, torch.float32), (12, 12, 64, torch.bfloat16),
                                           (9, 3, 256, torch.bfloat16)])
def test_bf16_results_of_small_groups(hip_backend, H, G, D, q_dtype, per_row):
    lens = [40 + 7 * (b % 11) for b in range(60)]
    got, want, tol = _run(hip_backend, rows(lens, H, G, D, 16, per_row, q_dtype), torch.bfloat16)
    assert int((~rounds_to(got, want, tol)).sum()) == 0


@pytest.mark.parametrize("per_row", [16, 128])
@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (16, 4, 128), (15, 5, 64), (7, 1, 128), (16, 2, 256), (5, 1, 64), (6, 1, 128)])
@pytest.mark.parametrize("q_dtype,spread", [(torch.float32, 1.0), (torch.float32, 6.0), (torch.bfloat16, 1.0)])
def test_f32_results(hip_backend, H, G, D, q_dtype, spread, per_row):
    q, *rest = rows([2, 5, 17, 40, 130, 200], H, G, D, 16, per_row, seed=H)
    got, want, tol = _run(hip_backend, [(q * spread).to(q_dtype), *rest], torch.float32)
    assert float(((got.double() - want).abs() / tol).max()) <= 1.0

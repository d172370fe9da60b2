"""Preparation over a paged cache: norm, rotary positions in both layouts, page writes."""

from __future__ import annotations

import pytest
import torch

from breezetoken_amd.backend import rope_tables, rope_tables_scaled
from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu


def _case(T, H, G, D, page, gated=True, norm=True, rope=None, cap=400, x_dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, H * D * (2 if gated else 1) + 2 * G * D, generator=g).to(x_dtype)
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)) if norm else (None, None)
    cos, sin = rope_tables(cap, rope, 1.0e4, "cpu") if rope else (None, None)
    rows = 3
    per_row = -(-cap // page)
    N = rows * per_row + 2
    table = torch.randperm(N, generator=g)[: rows * per_row].view(rows, per_row).to(torch.int32)
    slot = torch.randperm(rows * cap, generator=g)[:T]
    return qkv, wq, wk, cos, sin, (slot % cap).to(torch.int32), (slot // cap).to(torch.int32), table, N


def _check(be, c, H, G, D, page, gated, inter, rope, q_dtype=torch.float32, rows=True, eps=1e-6):
    qkv, wq, wk, cos, sin, pos, row, table, N = c
    g = torch.Generator().manual_seed(7)
    k0, v0 = (torch.randn(N, page, G, D, generator=g).to(torch.bfloat16) for _ in range(2))
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    k, v = k0.cuda(), v0.cuda()
    x = qkv.cuda()
    q, gate = be.attn_prep_paged(x, dev(wq), dev(wk), eps, dev(cos), dev(sin), pos.cuda(), rope or 0, k, v, table.cuda(), H,
                                 G, D, rows=row.cuda() if rows else None, gated=gated, interleaved=inter, q_dtype=q_dtype)
    rq, rk, rv, tq, tk = orc.prep(qkv, wq, wk, eps, cos, sin, pos, rope or 0, H, G, D, gated, inter)
    if q_dtype == torch.bfloat16:
        tq = tq + rq.abs() * orc.BF16 * 1.01
    assert bool(((q.double().cpu() - rq).abs() <= tq).all())
    if gated:
        assert torch.equal(gate.cpu(), qkv[:, : 2 * H * D].view(-1, H, 2 * D)[..., D:])
        assert gate.data_ptr() == x.data_ptr() + D * x.element_size()
    else:
        assert gate is None
    # Every other slot is as it was; v is rounded once, k to within its own error.
    wk_, wv_ = k0.clone(), v0.clone()
    per_row = table.shape[1]
    for t in range(len(pos)):
        r, p = int(row[t]) if rows else t, int(pos[t])
        if not (0 <= r < table.shape[0] and 0 <= p < per_row * page):
            continue
        i = int(table[r, p // page])
        if not 0 <= i < N:
            continue
        off = (k[i, p % page].double().cpu() - rk[t]).abs()
        assert bool((off <= tk[t] * 1.01 + rk[t].abs() * orc.BF16).all())
        wk_[i, p % page] = k[i, p % page].cpu()
        wv_[i, p % page] = rv[t].to(torch.bfloat16)
    assert torch.equal(wk_, k.cpu()) and torch.equal(wv_, v.cpu())


@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (32, 8, 128), (15, 5, 64), (7, 1, 128), (2, 1, 512), (1, 1, 64)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("gated,norm", [(True, True), (False, False), (False, True), (True, False)])
def test_shapes(hip_backend, H, G, D, inter, gated, norm):
    c = _case(37, H, G, D, 16, gated, norm, rope=D // 2)
    _check(hip_backend, c, H, G, D, 16, gated, inter, D // 2)


@pytest.mark.parametrize("rope", [2, 6, 10, 30, 32, 62, 64])
@pytest.mark.parametrize("inter", [False, True])
def test_part_of_the_head(hip_backend, rope, inter):
    _check(hip_backend, _case(20, 6, 2, 64, 16, rope=rope), 6, 2, 64, 16, True, inter, rope)
    _check(hip_backend, _case(20, 3, 1, 256, 16, rope=4 * rope), 3, 1, 256, 16, True, inter, 4 * rope)


@pytest.mark.parametrize("x_dtype,q_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                             (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_types(hip_backend, x_dtype, q_dtype, inter, D):
    c = _case(41, 4, 2, D, 32, False, True, rope=D, x_dtype=x_dtype)
    _check(hip_backend, c, 4, 2, D, 32, False, inter, D, q_dtype=q_dtype)


@pytest.mark.parametrize("T", [1, 2, 3, 64, 257, 1100])
@pytest.mark.parametrize("page", [16, 128, 1024])
def test_token_counts(hip_backend, T, page):
    _check(hip_backend, _case(T, 8, 2, 128, page, rope=128), 8, 2, 128, page, True, False, 128)


def test_no_rotation_and_rows_by_token(hip_backend):
    _check(hip_backend, _case(50, 4, 2, 128, 16), 4, 2, 128, 16, True, False, None)
    c = list(_case(3, 4, 2, 128, 16, rope=64))
    _check(hip_backend, c, 4, 2, 128, 16, True, False, 64, rows=False)


def test_tokens_without_a_slot_write_nothing(hip_backend):
    """Positions and rows outside the table, entries outside the cache; q is still given."""
    c = list(_case(40, 4, 2, 128, 16, rope=64, cap=200))
    pos, row, table = c[5], c[6], c[7]
    pos[:4] = torch.tensor([-1, 1 << 30, 13 * 16, -(1 << 31)], dtype=torch.int32)
    row[4:8] = torch.tensor([-1, 3, 1 << 30, -(1 << 31)], dtype=torch.int32)
    table[0, 2], table[1, 3], table[2, 0] = -1, c[8], 1 << 30
    _check(hip_backend, c, 4, 2, 128, 16, True, False, 64)


def test_zero_rows_and_large_values(hip_backend):
    c = _case(10, 4, 2, 128, 16, rope=128)
    c[0][0] = 0
    c[0][1] *= 1e15
    c[0][2] *= 1e-15
    _check(hip_backend, c, 4, 2, 128, 16, True, False, 128)


def test_strided_projection_and_cache(hip_backend):
    """qkv rows of a wider tensor, a misaligned one, and pages with heads before tokens."""
    T, H, G, D, page = 20, 4, 2, 128, 16
    qkv, wq, wk, cos, sin, pos, row, table, N = _case(T, H, G, D, page, rope=64)
    width = qkv.shape[1]
    args = lambda x, k, v: (x, wq.cuda(), wk.cuda(), 1e-6, cos.cuda(), sin.cuda(), pos.cuda(), 64, k, v, table.cuda(), H, G, D)  # noqa: E731
    pool = lambda: torch.zeros(N, page, G, D, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    k, v = pool(), pool()
    q, gate = hip_backend.attn_prep_paged(*args(qkv.cuda(), k, v), rows=row.cuda())
    for lead, trail in ((8, 16), (3, 2)):
        wide = torch.randn(T, lead + width + trail, device="cuda")
        wide[:, lead : lead + width] = qkv.cuda()
        k2 = torch.zeros(N, G, page, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        v2 = torch.zeros(N, G, page, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        q2, gate2 = hip_backend.attn_prep_paged(*args(wide[:, lead : lead + width], k2, v2), rows=row.cuda())
        assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(gate, gate2)


@pytest.mark.parametrize("method,trained", [("linear", None), ("ntk", None), ("yarn", 4096)])
def test_scaled_tables_at_far_positions(hip_backend, method, trained):
    cap, D = 65536, 128
    cos, sin = rope_tables_scaled(cap, D, 1.0e4, method, 8.0, trained, device="cpu")
    c = list(_case(9, 4, 2, D, 16, rope=D))
    c[3], c[4] = cos, sin
    c[5] = torch.tensor([0, 1, 4095, 4096, 32767, 65535, 399, 398, 70000], dtype=torch.int32)
    _check(hip_backend, c, 4, 2, D, 16, True, False, D)


def test_no_tokens(hip_backend):
    c = _case(1, 4, 2, 128, 16, rope=64)
    k = torch.zeros(c[8], 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    q, gate = hip_backend.attn_prep_paged(c[0][:0].cuda(), None, None, 1e-6, None, None, c[5][:0].cuda(), 0, k, k.clone(),
                                          c[7].cuda(), 4, 2, 128, rows=c[6][:0].cuda())
    assert q.shape == (0, 4, 128) and gate.shape == (0, 4, 128)


def test_agrees_with_the_single_token_preparation(hip_backend):
    """One token of the contiguous path and of the paged one: the same q, k and v."""
    H, G, D = 8, 2, 256
    qkv, wq, wk, cos, sin, *_ = (None if t is None else t.cuda() for t in _case(1, H, G, D, 16, rope=64)[:5] + (None,))
    pos = torch.tensor([37], dtype=torch.int32, device="cuda")
    ck, cv = (torch.zeros(64, G, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q1, gate1 = hip_backend.attn_prep(qkv[0], wq, wk, 1e-6, cos, sin, pos, 64, ck, cv, H, G, D)
    pk, pv = (torch.zeros(4, 16, G, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    q2, gate2 = hip_backend.attn_prep_paged(qkv, wq, wk, 1e-6, cos, sin, pos, 64, pk, pv, table, H, G, D)
    assert float((q1 - q2[0]).abs().max()) <= 32 * orc.F32 * float(q1.abs().max()) and torch.equal(gate1, gate2[0])
    assert torch.equal(cv, pv.view_as(cv))
    assert float((ck.float() - pk.view_as(ck).float()).abs().max()) <= 2 * orc.BF16 * float(ck.float().abs().max())

"""The paged operators called at once: on streams of their own, from threads, in graphs
replayed side by side; results are those of a call alone, which other tests check."""

from __future__ import annotations

import threading

import pytest
import torch

from breezetoken_amd.backend import rope_tables
from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu

PAGE = 16


def _prep(be, seed):
    g = torch.Generator().manual_seed(seed)
    T, H, G, D = 40 + seed, 8, 2, 128
    qkv = torch.randn(T, (2 * H + 2 * G) * D, generator=g).cuda()
    w = torch.rand(D, generator=g).cuda()
    cos, sin = rope_tables(200, 64, 10000.0, "cuda")
    pos, rows = torch.arange(T, dtype=torch.int32).cuda(), torch.zeros(T, dtype=torch.int32).cuda()
    table = torch.randperm(6, generator=g).view(1, 6).to(torch.int32).cuda()
    k, v = (torch.zeros(6, PAGE, G, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def call():
        q, _ = be.attn_prep_paged(qkv, w, w, 1e-6, cos, sin, pos, 64, k, v, table, H, G, D, rows=rows)
        return q, k, v

    return call


def _tables(seed, rows=7, pages=60, per_row=8):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, per_row * PAGE - 20, (rows,), generator=g, dtype=torch.int32)
    return orc.page_table(lens.tolist(), PAGE, per_row, pages, seed).cuda(), lens.cuda()


def _fork(be, seed):
    """Room for tokens in a pool that a call leaves as it was: no page is shared and written."""
    table, lens = _tables(seed)
    pool = torch.randn(2, 60, PAGE, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    return lambda: be.fork_pages(pool, table, lens, add=3 + seed) + (pool,)


def _compact(be, seed):
    """A pool that is tidy already: a call moves nothing."""
    table, lens = _tables(seed)
    pool = torch.randn(2, 60, PAGE, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    table, _, _ = be.compact_pages(pool, table, lens)
    return lambda: be.compact_pages(pool, table, lens) + (pool,)


def _beam(be, seed):
    g = torch.Generator().manual_seed(seed)
    logits, scores = torch.randn(3, 4, 9000 + seed, generator=g).cuda(), torch.randn(3, 4, generator=g).cuda()
    return lambda: be.beam_select(logits, scores)


OPS = [_prep, _fork, _compact, _beam]


def _alone(call):
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    return want


def _equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


@pytest.mark.parametrize("make", OPS)
def test_two_streams_at_once(hip_backend, make):
    calls = [make(hip_backend, s) for s in (0, 1)]
    want = [_alone(c) for c in calls]
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    for _ in range(8):
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(c())
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(_equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("make", OPS)
def test_threads_call_at_once(hip_backend, make):
    calls = [make(hip_backend, s) for s in range(4)]
    want = [_alone(c) for c in calls]
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                got = calls[i]()
                torch.cuda.current_stream().synchronize()
                if not _equal(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("make", OPS)
def test_two_graphs_replayed_side_by_side(hip_backend, make):
    calls = [make(hip_backend, s) for s in (0, 1)]
    want = [_alone(c) for c in calls]
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c in calls:
            c()  # eager work between the replays
        torch.cuda.synchronize()
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(_equal(outs[i], want[i]) for i in (0, 1))


def test_operands_at_odd_offsets(hip_backend):
    """Contiguous tensors whose first value is not aligned to 16 bytes."""
    g = torch.Generator().manual_seed(0)
    H, G, D, B = 8, 2, 128, 3
    k, v = (torch.randn(12, PAGE, G, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    table = torch.randperm(12, generator=g).view(B, 4).to(torch.int32).cuda()
    lens = torch.tensor([60, 1, 17], dtype=torch.int32).cuda()
    q = torch.randn(B, H, D, generator=g).cuda()
    odd = torch.empty(q.numel() + 1, device="cuda")[1:].view(B, H, D).copy_(q)
    assert odd.data_ptr() % 16
    assert torch.equal(hip_backend.attention_paged(odd, k, v, table, lens, 0.1),
                       hip_backend.attention_paged(q, k, v, table, lens, 0.1))
    qkv = torch.randn(B, (2 * H + 2 * G) * D, generator=g).cuda()
    odd = torch.empty(qkv.numel() + 1, device="cuda")[1:].view(qkv.shape).copy_(qkv)
    pos = torch.tensor([59, 0, 16], dtype=torch.int32).cuda()
    got = []
    for x in (qkv, odd):
        k1, v1 = k.clone(), v.clone()
        y, gate = hip_backend.attn_prep_paged(x, None, None, 0.0, None, None, pos, 0, k1, v1, table, H, G, D)
        got.append((y, gate.clone(), k1, v1))
    assert _equal(got[0], got[1])


def test_rows_that_ask_for_more_than_any_table(hip_backend):
    """The pages that cannot be given are more than 31 bits count: still a positive number."""
    table, lens = _tables(3, rows=70, pages=600)
    pool = torch.zeros(2, 600, PAGE, 64, dtype=torch.bfloat16, device="cuda")
    add = torch.full((70,), 2**31 - 1, dtype=torch.int32, device="cuda")
    new, kept, status = hip_backend.fork_pages(pool, table, lens, add=add)
    assert torch.equal(kept, lens)
    assert int(status[1]) == 70 * ((1 << 30) // 70)  # the pool itself suffices: 70 rows of 8
    used = -(-lens // PAGE)
    held = torch.arange(8, device="cuda")[None] < used[:, None]
    assert torch.equal(new[held], table[held]) and int((new >= 0).sum()) == 70 * 8


@pytest.mark.parametrize("B,W", [(300, 4), (1100, 2), (2100, 3)])
def test_more_rows_than_waves_are_wanted(hip_backend, B, W):
    g = torch.Generator().manual_seed(B)
    logits, scores = torch.randn(B, W, 4200, generator=g) * 3, -torch.rand(B, W, generator=g)
    got = hip_backend.beam_select(logits.cuda(), scores.cuda())
    want = orc.beams(logits, scores, W)
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])
    assert bool(((got[0].cpu().double() - want[0]).abs() <= want[0].abs() * orc.F32 + 2.0**-22).all())

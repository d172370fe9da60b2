"""Decode attention over a paged cache against 64-bit attention over the same keys."""

from __future__ import annotations

import pytest
import torch

from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu


def _case(lens, H, G, D, page, per_row=None, q_dtype=torch.float32, seed=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    per_row = per_row or max(1, -(-max(list(lens) + [1]) // page) + 1)
    N = sum(-(-n // page) for n in lens) + spare
    k = torch.randn(N, page, G, D, generator=g).to(torch.bfloat16)
    v = torch.randn(N, page, G, D, generator=g).to(torch.bfloat16)
    q = torch.randn(len(lens), H, D, generator=g).to(q_dtype)
    return q, k, v, orc.page_table(lens, page, per_row, N, seed), torch.tensor(lens, dtype=torch.int32)


def _check(be, q, k, v, table, lens, out_dtype=torch.float32, ref=None, got=None):
    scale = q.shape[-1] ** -0.5
    if ref is None:
        ref = orc.attention(q, k, v, table, lens, scale)
    if got is None:
        got = be.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), scale, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    tol = orc.attention_tolerance(q, k, v, scale, max(1, int(lens.max()) if lens.numel() else 1), ref,
                                  out_dtype == torch.bfloat16)
    off = (got.double().cpu() - ref).abs()
    assert bool((off <= tol).all()), (float(off.max()), float(tol.max()))
    return ref


@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (16, 2, 256), (32, 8, 128), (12, 12, 64), (15, 5, 64), (7, 1, 128), (5, 1, 256)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                               (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_shapes_and_types(hip_backend, H, G, D, q_dtype, out_dtype):
    _check(hip_backend, *_case([1, 37, 301, 16, 130], H, G, D, 32, q_dtype=q_dtype), out_dtype=out_dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 255, 256, 257, 1025])
def test_lengths_around_pages(hip_backend, page, length):
    _check(hip_backend, *_case([length], 8, 2, 128, page))


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [0, 5, 0, 700, 0], [3, 0], [0, 1]])
def test_rows_without_tokens_are_zero(hip_backend, lens):
    q, k, v, table, n = _case(lens, 8, 2, 256, 16)
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), 0.0625)
    _check(hip_backend, q, k, v, table, n, got=got)
    assert not got.cpu()[[i for i, x in enumerate(lens) if x == 0]].any()


@pytest.mark.parametrize("batch", [1, 2, 33, 130, 300])
def test_ragged_batches(hip_backend, batch):
    g = torch.Generator().manual_seed(batch)
    lens = [int(x) for x in torch.exp(torch.rand(batch, generator=g) * 6.5)]
    _check(hip_backend, *_case(lens, 8, 2, 64, 16, seed=batch))


@pytest.mark.parametrize("H,G,D,length", [(8, 2, 256, 20001), (16, 2, 128, 9000)])
def test_long_rows(hip_backend, H, G, D, length):
    _check(hip_backend, *_case([length, 3], H, G, D, 64))


def test_wide_table_and_largest_batch(hip_backend):
    # A table for far more tokens than there are, and the most sequences a call takes.
    _check(hip_backend, *_case([100, 1, 40], 8, 2, 128, 16, per_row=9000))
    lens = [b % 3 for b in range(4096)]
    _check(hip_backend, *_case(lens, 2, 1, 64, 16, per_row=2))


def test_lengths_outside_the_row_are_clamped(hip_backend):
    q, k, v, table, lens = _case([64, 64, 20], 8, 2, 128, 16, per_row=4)
    lens = torch.tensor([1 << 30, -7, 20], dtype=torch.int32)
    clamped = torch.tensor([64, 0, 20], dtype=torch.int32)
    ref = orc.attention(q, k, v, table, clamped, 128**-0.5)
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), 128**-0.5)
    _check(hip_backend, q, k, v, table, clamped, ref=ref, got=got)


def test_entries_outside_the_cache_hold_no_keys(hip_backend):
    q, k, v, table, lens = _case([200, 50, 16, 100], 8, 2, 128, 16)
    table[0, 3], table[0, 12] = -1, k.shape[0]
    table[1, 0] = 1 << 30
    table[2, 0] = -(1 << 31)
    _check(hip_backend, q, k, v, table, lens)


def test_slots_without_tokens_are_not_read(hip_backend):
    """NaN and infinities in free pages, and behind the last token of a page."""
    lens = [5, 33, 48, 250]
    q, k, v, table, n = _case(lens, 8, 2, 256, 16, spare=8)
    ref = orc.attention(q, k, v, table, n, 0.0625)
    live = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, length in enumerate(lens):
        for t in range(length):
            live[table[b, t // 16], t % 16] = True
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
    fill = bad[torch.randint(0, 4, k.shape, generator=torch.Generator().manual_seed(9))].to(torch.bfloat16)
    k2, v2 = torch.where(live[..., None, None], k, fill), torch.where(live[..., None, None], v, fill)
    got = hip_backend.attention_paged(q.cuda(), k2.cuda(), v2.cuda(), table.cuda(), n.cuda(), 0.0625)
    _check(hip_backend, q, k, v, table, n, ref=ref, got=got)


def test_a_nan_query_or_key_gives_nan(hip_backend):
    q, k, v, table, n = _case([100, 100], 8, 2, 128, 16)
    q[0, 3, 5] = float("nan")
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), 0.1).cpu()
    assert got[0, 3].isnan().all() and got[1].isfinite().all() and got[0, :3].isfinite().all()


def test_large_scores(hip_backend):
    """Scores of hundreds: the softmax keeps one or few keys."""
    q, k, v, table, n = _case([300, 17], 8, 2, 128, 32)
    _check(hip_backend, q * 40, k, v, table, n)
    q[:] = -30.0
    k[:] = k.abs()  # every score far below zero
    _check(hip_backend, q, k, v, table, n)


def test_shared_pages(hip_backend):
    """One page in several rows, and twice in one."""
    q, k, v, table, n = _case([64, 40, 64], 8, 2, 128, 16)
    table[1, :2] = table[0, :2]
    table[2, 3] = table[2, 0]
    _check(hip_backend, q, k, v, table, n)


def test_strided_caches_and_queries(hip_backend):
    """Heads before tokens in a page, one plane of many, q of a fused projection."""
    q, k, v, table, n = _case([100, 31], 8, 2, 128, 32)
    ref = orc.attention(q, k, v, table, n, 128**-0.5)
    by_head = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v)]
    got = hip_backend.attention_paged(q.cuda(), *by_head, table.cuda(), n.cuda(), 128**-0.5)
    _check(hip_backend, q, k, v, table, n, ref=ref, got=got)
    both = torch.stack((k, v), dim=1).cuda()  # (N, 2, page, G, D): K and V of a page side by side
    wide = torch.randn(2, 20, 128)
    wide[:, 4:12] = q
    got = hip_backend.attention_paged(wide.cuda()[:, 4:12], both[:, 0], both[:, 1], table.cuda(), n.cuda(), 128**-0.5)
    _check(hip_backend, q, k, v, table, n, ref=ref, got=got)


def test_cache_past_32_bit_offsets(hip_backend):
    """A plane of 5 GiB: pages whose first element lies past 2^31 and 2^32 bytes."""
    page, G, D, N = 256, 2, 256, 20500
    k = torch.zeros(N, page, G, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(N, page, G, D, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(3)
    ids = torch.tensor([[N - 1, 0, 8192, 16384], [4096, N - 2, 12288, 5]], dtype=torch.int32)
    small_k = torch.randn(8, page, G, D, generator=g).to(torch.bfloat16)
    small_v = torch.randn(8, page, G, D, generator=g).to(torch.bfloat16)
    k[ids.flatten().long()], v[ids.flatten().long()] = small_k.cuda(), small_v.cuda()
    q = torch.randn(2, 8, D, generator=g)
    lens = torch.tensor([1000, 700], dtype=torch.int32)
    got = hip_backend.attention_paged(q.cuda(), k, v, ids.cuda(), lens.cuda(), 0.0625)
    _check(hip_backend, q, small_k, small_v, torch.arange(8, dtype=torch.int32).view(2, 4), lens, got=got)


def test_repeated_calls_are_equal(hip_backend):
    args = [t.cuda() for t in _case([3000, 17, 900], 8, 2, 256, 32)]
    first = hip_backend.attention_paged(*args, 0.0625)
    for _ in range(3):
        assert torch.equal(first, hip_backend.attention_paged(*args, 0.0625))


def test_two_streams_at_once(hip_backend):
    a = [t.cuda() for t in _case([5000, 17], 8, 2, 256, 32, seed=1)]
    b = [t.cuda() for t in _case([40, 4000, 9], 8, 2, 256, 32, seed=2)]
    want = hip_backend.attention_paged(*a, 0.0625), hip_backend.attention_paged(*b, 0.0625)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(10):
        for i, args in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(hip_backend.attention_paged(*args, 0.0625))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_captured_with_growing_lengths(hip_backend):
    """One graph, replayed as the sequences grow; two graphs of different shapes side by side."""
    q, k, v, table, lens = (t.cuda() for t in _case([600, 100, 1], 8, 2, 128, 16, per_row=45, spare=80))
    table.copy_(torch.randperm(table.numel(), generator=torch.Generator().manual_seed(5)).view_as(table) % k.shape[0])
    other = [t.cuda() for t in _case([2000], 8, 2, 128, 32)]
    scale = 128**-0.5
    for args in ((q, k, v, table, lens), other):  # warm up
        hip_backend.attention_paged(*args, scale)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        out = hip_backend.attention_paged(q, k, v, table, lens, scale)
    with torch.cuda.graph(second):
        out2 = hip_backend.attention_paged(*other, scale)
    want2 = hip_backend.attention_paged(*other, scale)
    for grown in ([600, 100, 1], [601, 116, 2], [720, 0, 17], [3, 720, 720]):
        lens.copy_(torch.tensor(grown, dtype=torch.int32))
        first.replay()
        second.replay()
        eager = hip_backend.attention_paged(q, k, v, table, lens, scale)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(out2, want2)
        _check(hip_backend, q.cpu(), k.cpu(), v.cpu(), table.cpu(), lens.cpu(), got=out)


WIDE = 1024  # tokens a table row has room for: the work is split into runs, at most a work-group each


def _wide(lens, H, G, D, page, **kw):
    return _case(lens, H, G, D, page, per_row=WIDE // page, **kw)


@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (15, 5, 64), (7, 1, 128), (16, 4, 128), (4, 1, 256)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                               (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_runs_shapes_and_types(hip_backend, H, G, D, q_dtype, out_dtype):
    _check(hip_backend, *_wide([1, 37, 1024, 16, 130, 513], H, G, D, 32, q_dtype=q_dtype), out_dtype=out_dtype)


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [0, 5, 0, 700, 0], [3, 0], [0, 1], [1024], [1023, 1, 1024],
                                  [16] * 70, [0] * 65 + [1] + [0] * 64, [17, 0] * 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_runs_with_rows_without_tokens(hip_backend, lens, D):
    q, k, v, table, n = _wide(lens, 8, 2, D, 16)
    scale = D**-0.5
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), scale)
    _check(hip_backend, q, k, v, table, n, got=got)
    assert not got.cpu()[[i for i, x in enumerate(lens) if x == 0]].any()


@pytest.mark.parametrize("batch", [63, 64, 65, 512, 513, 700, 4096])
def test_runs_over_many_sequences(hip_backend, batch):
    """Windows of 64 lengths, the first eight of them kept."""
    g = torch.Generator().manual_seed(batch)
    lens = [int(x) for x in torch.exp(torch.rand(batch, generator=g) * 4.0) - 1.0]
    lens[batch // 2] = 900
    _check(hip_backend, *_wide(lens, 2, 1, 64, 16, seed=batch))


def test_runs_lengths_outside_the_row_are_clamped(hip_backend):
    q, k, v, table, lens = _wide([1024, 64, 20], 8, 2, 128, 16)
    lens = torch.tensor([(1 << 31) - 1, -(1 << 31), 20], dtype=torch.int32)
    clamped = torch.tensor([1024, 0, 20], dtype=torch.int32)
    ref = orc.attention(q, k, v, table, clamped, 128**-0.5)
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), 128**-0.5)
    _check(hip_backend, q, k, v, table, clamped, ref=ref, got=got)


def test_runs_entries_outside_the_cache_hold_no_keys(hip_backend):
    q, k, v, table, lens = _wide([200, 50, 16, 1000], 8, 2, 128, 16)
    table[0, 3], table[0, 12] = -1, k.shape[0]
    table[1, 0] = 1 << 30
    table[2, 0] = -(1 << 31)  # its only entry: no keys at all
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), 128**-0.5)
    _check(hip_backend, q, k, v, table, lens, got=got)
    assert not got[2].any()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_runs_do_not_read_slots_without_tokens(hip_backend, D):
    lens = [5, 33, 48, 250, 1001]
    q, k, v, table, n = _wide(lens, 8, 2, D, 64, spare=8)
    ref = orc.attention(q, k, v, table, n, 0.0625)
    live = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, length in enumerate(lens):
        for t in range(length):
            live[table[b, t // 64], t % 64] = True
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
    fill = bad[torch.randint(0, 4, k.shape, generator=torch.Generator().manual_seed(9))].to(torch.bfloat16)
    k2, v2 = torch.where(live[..., None, None], k, fill), torch.where(live[..., None, None], v, fill)
    got = hip_backend.attention_paged(q.cuda(), k2.cuda(), v2.cuda(), table.cuda(), n.cuda(), 0.0625)
    tol = orc.attention_tolerance(q, k, v, 0.0625, 1001, ref, False)
    assert bool(((got.double().cpu() - ref).abs() <= tol).all())


def test_runs_nan_query(hip_backend):
    q, k, v, table, n = _wide([1000, 100], 8, 2, 128, 16)
    q[0, 3, 5] = float("nan")
    got = hip_backend.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), 0.1).cpu()
    assert got[0, 3].isnan().all() and got[1].isfinite().all() and got[0, :3].isfinite().all()


def test_runs_large_scores_and_shared_pages(hip_backend):
    q, k, v, table, n = _wide([900, 17, 640], 8, 2, 128, 32)
    table[2, :20] = table[0, :20]
    table[2, 3] = table[2, 0]
    _check(hip_backend, q * 40, k, v, table, n)
    q[:] = -30.0
    k[:] = k.abs()  # every score far below zero
    _check(hip_backend, q, k, v, table, n)


def test_a_sequence_does_not_change_with_its_batch_in_whole_mode(hip_backend):
    """Short tables: a work-group takes a sequence, so its bits depend on nothing else."""
    q, k, v, table, n = (t.cuda() for t in _case([300, 7, 512, 0, 64], 8, 2, 128, 16, per_row=32))
    got = hip_backend.attention_paged(q, k, v, table, n, 0.1)
    for b in range(5):
        alone = hip_backend.attention_paged(q[b : b + 1], k, v, table[b : b + 1], n[b : b + 1], 0.1)
        assert torch.equal(alone[0], got[b])


def test_on_another_stream_than_the_current_one(hip_backend):
    """Tensors made on one stream, used on a second that waits for it, freed while in flight."""
    side = torch.cuda.Stream()
    want = None
    for _ in range(4):
        args = [t.cuda() for t in _wide([1000, 40, 3], 8, 2, 256, 32)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = hip_backend.attention_paged(*args, 0.0625)
        for t in args:
            t.record_stream(side)
        del args
        side.synchronize()
        want = got if want is None else want
        assert torch.equal(got, want)


def test_two_graphs_replayed_in_turn_and_on_two_streams(hip_backend):
    a = [t.cuda() for t in _wide([1000, 17], 8, 2, 256, 32, seed=1)]
    b = [t.cuda() for t in _wide([40, 900, 9], 8, 2, 256, 32, seed=2)]
    want = hip_backend.attention_paged(*a, 0.0625), hip_backend.attention_paged(*b, 0.0625)
    graphs, outs = [], []
    for args in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(hip_backend.attention_paged(*args, 0.0625))
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for i in (0, 1):
            outs[i].zero_()
        torch.cuda.synchronize()
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_threads_call_at_once(hip_backend):
    """Four threads, a stream and shapes of their own each; every result is the one alone."""
    import threading

    cases = [[t.cuda() for t in _wide([700 + 50 * i, 20, 0, 333], 8, 2, 128, 16, seed=i)] for i in range(4)]
    want = [hip_backend.attention_paged(*c, 0.1) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = hip_backend.attention_paged(*cases[i], 0.1)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("batch", [65, 512, 513, 700, 4096])
def test_runs_over_many_sequences_of_long_tables(hip_backend, batch):
    """Room for 2,048 tokens a row: runs for any number of sequences, windows of their lengths past the eighth."""
    g = torch.Generator().manual_seed(batch)
    lens = [int(x) for x in torch.exp(torch.rand(batch, generator=g) * 4.0) - 1.0]
    lens[batch // 2] = 2048
    lens[batch - 1] = 700
    _check(hip_backend, *_case(lens, 2, 1, 64, 16, per_row=128, seed=batch))


@pytest.mark.parametrize("H,G,D,batch", [(8, 2, 256, 128), (8, 2, 256, 127), (32, 8, 128, 32), (15, 5, 64, 60)])
def test_sequences_that_fill_the_chip(hip_backend, H, G, D, batch):
    """A work-group per sequence up to 1,024 tokens, and a batch that is one short of that."""
    g = torch.Generator().manual_seed(batch)
    lens = [int(x) for x in torch.exp(torch.rand(batch, generator=g) * 6.9)]
    lens[0], lens[5], lens[batch - 1] = 1024, 0, 1023
    _check(hip_backend, *_case(lens, H, G, D, 64, per_row=16, seed=batch))


def test_no_sequences(hip_backend):
    q, k, v, table, lens = _case([3], 8, 2, 128, 16)
    got = hip_backend.attention_paged(q[:0].cuda(), k.cuda(), v.cuda(), table[:0].cuda(), lens[:0].cuda(), 0.1)
    assert got.shape == (0, 8, 128)

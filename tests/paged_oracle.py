"""Plain 64-bit (and plain integer) forms of the paged cache's operators, for the tests."""

from __future__ import annotations

import math

import torch

F32, BF16 = 2.0**-24, 2.0**-8  # half a step of each type, relative


def page_table(lens, page: int, per_row: int, num_pages: int, seed: int = 0) -> torch.Tensor:
    """A table whose rows own their pages, ids in random order; unused entries hold ids of other rows."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(num_pages, generator=g).to(torch.int32)
    table = torch.randint(0, num_pages, (len(lens), per_row), generator=g, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = ids[at : at + m]
        at += m
    assert at <= num_pages
    return table


def attention(q, k, v, table, lens, scale: float) -> torch.Tensor:
    """(B, H, D) in 64 bits; entries outside the cache hold no keys."""
    q, k, v = q.double(), k.double(), v.double()
    B, H, D = q.shape
    N, page, G, _ = k.shape
    out = torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        slots = [(int(table[b, t // page]), t % page) for t in range(max(0, min(int(lens[b]), table.shape[1] * page)))]
        slots = [(i, t) for i, t in slots if 0 <= i < N]
        if not slots:
            continue
        ids, at = torch.tensor([s[0] for s in slots]), torch.tensor([s[1] for s in slots])
        for g in range(G):
            x = q[b, g * (H // G) : (g + 1) * (H // G)] @ k[ids, at, g].T * scale
            out[b, g * (H // G) : (g + 1) * (H // G)] = torch.softmax(x, dim=1) @ v[ids, at, g]
    return out


def attention_tolerance(q, k, v, scale: float, keys: int, out: torch.Tensor, bf16_out: bool) -> torch.Tensor:
    """What f32 scores and sums may be off, elementwise over ``out``.

    A score sums D products in f32: at most sqrt(D) + 8 half steps of sum |q k|
    (steps of random sign; the worst case would be D), and its exponential has
    another few.  A probability off by a factor e^d moves the output by at most
    2 d max|v|.  The weighted sum over the keys adds sqrt(keys) + 32 half steps of
    max|v|.  Where the output is bf16, q and the probabilities may enter as two
    bf16 terms, which leave 2^-16 of each."""
    D = q.shape[-1]
    reach = q.double().abs().amax() * k.double().abs().amax() * scale * math.sqrt(D) * 2
    top = float(v.double().abs().amax())
    d = float(reach) * (math.sqrt(D) + 8) * F32 + 8 * F32
    tol = top * (2 * d + (math.sqrt(keys) + 32) * F32)
    if bf16_out:
        tol += top * 2 * (float(reach) + 1) * BF16**2
        return tol + out.abs() * BF16
    return torch.full_like(out, tol)


def prep(qkv, wq, wk, eps, cos, sin, pos, rope: int, H: int, G: int, D: int, gated: bool, inter: bool):
    """q, k, v (T, heads, D) in 64 bits, and what f32 arithmetic may be off in q and k."""
    x = qkv.double()
    T, step = x.shape[0], (2 * D if gated else D)
    q = x[:, : H * step].reshape(T, H, step)[..., :D].clone()
    k = x[:, H * step : H * step + G * D].reshape(T, G, D).clone()
    v = x[:, H * step + G * D :].reshape(T, G, D)
    tol = []
    for t, w in ((q, wq), (k, wk)):
        # The mean square's sum, its root, its inverse and two products: 16 half steps.
        if w is not None:
            t.mul_(torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * w.double())
        off = t.abs() * 16 * F32
        if cos is not None:
            i = torch.arange(rope // 2)
            a, b = (2 * i, 2 * i + 1) if inter else (i, i + rope // 2)
            row = pos.long().clamp(0, cos.shape[0] - 1)
            c, s = cos[row][:, None, : rope // 2].double(), sin[row][:, None, : rope // 2].double()
            ta, tb = t[..., a].clone(), t[..., b].clone()
            t[..., a], t[..., b] = ta * c - tb * s, tb * c + ta * s
            both = (ta.abs() + tb.abs()) * torch.maximum(c.abs(), s.abs()) * 20 * F32
            off[..., a], off[..., b] = both, both
        tol.append(off)
    return q, k, v, tol[0], tol[1]


def fork(pages, table, lens, parent, add, keep=()):
    """(table, lens, status, pages) by the definition, one row after the other."""
    pages, before = pages.clone(), pages
    N, page, P = pages.shape[1], pages.shape[2], table.shape[1]
    rows_in = table.shape[0]
    rows, new_lens, held = [], [], [0] * N
    for p in parent:
        n = min(max(int(lens[p]), 0), P * page) if 0 <= p < rows_in else 0
        row = [int(i) if 0 <= int(i) < N else -1 for i in (table[p][: -(-n // page)] if n else [])]
        rows.append(row)
        new_lens.append(n)
        for i in row:
            if i >= 0:
                held[i] += 1
    for i in keep:
        if 0 <= i < N:
            held[i] += 1
    free = [i for i in range(N) if held[i] == 0]
    missing = 0
    for row, n, a in zip(rows, new_lens, add):
        a = max(int(a), 0)
        if a and n % page and row[-1] >= 0 and held[row[-1]] > 1:
            if free:
                to = free.pop(0)
                pages[:, to, : n % page] = before[:, row[-1], : n % page]
                row[-1] = to
            else:
                row[-1] = -1
                missing += 1
        need = -(-(n + a) // page)
        missing += max(0, need - P)
        while len(row) < min(need, P):
            if free:
                row.append(free.pop(0))
            else:
                row.append(-1)
                missing += 1
    out = torch.full((len(rows), P), -1, dtype=torch.int32)
    for i, row in enumerate(rows):
        out[i, : len(row)] = torch.tensor(row, dtype=torch.int32)
    return out, torch.tensor(new_lens, dtype=torch.int32), torch.tensor([len(free), missing], dtype=torch.int32), pages


def compact(pages, table, lens, keep=()):
    pages, before = pages.clone(), pages
    N, page, P = pages.shape[1], pages.shape[2], table.shape[1]
    rows = []
    for b in range(table.shape[0]):
        n = min(max(int(lens[b]), 0), P * page)
        rows.append([int(i) if 0 <= int(i) < N else -1 for i in table[b][: -(-n // page)]])
    live = sorted({i for row in rows for i in row if i >= 0} | {i for i in keep if 0 <= i < N})
    holes = [i for i in range(len(live)) if i not in set(live)]
    where = torch.full((N,), -1, dtype=torch.int32)
    for i in live:
        where[i] = i if i < len(live) else holes.pop(0)
        if where[i] != i:
            pages[:, int(where[i])] = before[:, i]
    out = torch.full_like(table, -1)
    for b, row in enumerate(rows):
        for c, i in enumerate(row):
            out[b, c] = where[i] if i >= 0 else -1
    return out, where, torch.tensor([len(live)], dtype=torch.int32), pages


def beams(logits, scores, count: int):
    """(scores in 64 bits, parent, token) by sorting every candidate."""
    B, W, V = logits.shape
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    best, parent, token = [], [], []
    for b in range(B):
        found = []
        for w in range(W):
            # Relative to the largest first: logits of 1e38 would swallow the log of the sum in 64 bits too.
            top = x[b, w].max()
            c = (x[b, w] - top) - torch.log(torch.exp(x[b, w] - top).sum()) + float(scores[b, w])
            c = torch.where(c.isnan(), -math.inf, c)
            xs = x[b, w].tolist()
            order = sorted(range(V), key=lambda t: (-xs[t], t))[:count]
            found += [(-float(c[t]), w, i, t) for i, t in enumerate(order)]
        found = sorted(found)[:count]
        best.append([-f[0] for f in found])
        parent.append([b * W + f[1] for f in found])
        token.append([f[3] for f in found])
    return torch.tensor(best, dtype=torch.float64), torch.tensor(parent), torch.tensor(token)

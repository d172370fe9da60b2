"""The paged cache's operators together: prompts into pages, then a beam search whose
sequences share them, against a model that keeps every sequence's history apart."""

from __future__ import annotations

import pytest
import torch

from breezetoken_amd import PagedKVCache
from breezetoken_amd.backend import rope_tables
from tests import paged_oracle as orc

pytestmark = pytest.mark.gpu

H, G, D, LAYERS, E, V, PAGE, ROPE = 4, 2, 128, 2, 64, 500, 16, 64
SCALE, EPS = D**-0.5, 1e-6


class Model:
    def __init__(self, seed: int) -> None:
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.emb = r(V, E)
        self.wqkv = [r(E, 2 * H * D + 2 * G * D) / 8 for _ in range(LAYERS)]
        self.wo = [r(H * D, E) / 22 for _ in range(LAYERS)]
        self.norms = [(1 + 0.1 * r(D), 1 + 0.1 * r(D)) for _ in range(LAYERS)]
        self.head = r(E, V) / 4
        self.cos, self.sin = rope_tables(256, ROPE, 1.0e4, "cpu")

    def cuda(self):
        for name in ("emb", "head", "cos", "sin"):
            setattr(self, name, getattr(self, name).cuda())
        self.wqkv, self.wo = [t.cuda() for t in self.wqkv], [t.cuda() for t in self.wo]
        self.norms = [(a.cuda(), b.cuda()) for a, b in self.norms]
        return self

    def plain_logits(self, tokens: list[int]) -> torch.Tensor:
        """Next-token logits in 64 bits over a whole history; keys and values rounded to bf16 as a cache holds them."""
        x = self.emb[torch.tensor(tokens)].double()
        T = x.shape[0]
        causal = torch.ones(T, T).tril().bool()
        for i in range(LAYERS):
            qkv = x @ self.wqkv[i].double()
            q, k, v, _, _ = orc.prep(qkv, *self.norms[i], EPS, self.cos, self.sin, torch.arange(T), ROPE, H, G, D, True, False)
            k, v = k.to(torch.bfloat16).double(), v.to(torch.bfloat16).double()
            out = torch.zeros(T, H, D, dtype=torch.float64)
            for h in range(H):
                s = (q[:, h] @ k[:, h // (H // G)].T * SCALE).masked_fill(~causal, float("-inf"))
                out[:, h] = torch.softmax(s, 1) @ v[:, h // (H // G)]
            gate = qkv[:, : 2 * H * D].view(T, H, 2 * D)[..., D:]
            x = x + (out * torch.sigmoid(gate)).reshape(T, -1) @ self.wo[i].double()
        return x[-1] @ self.head.double()


def _layer(be, m, i, x, pos, rows, cache, table, attend):
    qkv = x @ m.wqkv[i]
    k, v = cache.layer(i)
    q, gate = be.attn_prep_paged(qkv, *m.norms[i], EPS, m.cos, m.sin, pos, ROPE, k, v, table, H, G, D, rows=rows)
    out = attend(i, q, k, v)
    return x + (out * torch.sigmoid(gate)).reshape(x.shape[0], -1) @ m.wo[i]


def _prompt(be, m, cache, prompts, max_tokens):
    """Prompts into a fresh cache: their pages are consecutive, so prompt attention reads them as flat rows."""
    table, lens = cache.empty_table(len(prompts), max_tokens)
    sizes = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    table, lens, status = be.fork_pages(cache.pages, table, lens, add=sizes)
    first = table[:, 0].tolist()
    logits = []
    for b, p in enumerate(prompts):
        x = m.emb[torch.tensor(p, device="cuda")]
        pos = torch.arange(len(p), dtype=torch.int32, device="cuda")
        attend = lambda i, q, k, v: be.attention_prefill(q, *cache.rows(i, first[b], len(p)), SCALE)  # noqa: B023, E731
        for i in range(LAYERS):
            x = _layer(be, m, i, x, pos, torch.full_like(pos, b), cache, table, attend)
        logits.append(x[-1] @ m.head)
    return table, sizes, torch.stack(logits), status


def _step(be, m, cache, token, table, lens):
    """Logits behind one more token per row; the rows' pages have room for it."""
    x = m.emb[token.long()]
    now = lens + 1
    attend = lambda i, q, k, v: be.attention_paged(q, k, v, table, now, SCALE)  # noqa: E731
    for i in range(LAYERS):
        x = _layer(be, m, i, x, lens, None, cache, table, attend)
    return x @ m.head, now


@pytest.mark.parametrize("W,lengths", [(3, (21, 16)), (5, (1, 47, 32)), (1, (9,))])
def test_beam_search_over_shared_pages(hip_backend, W, lengths):
    be, m = hip_backend, Model(W)
    g = torch.Generator().manual_seed(W)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in lengths]
    B, steps = len(prompts), 20
    plain, m = m, Model(W).cuda()
    cache = PagedKVCache(160, PAGE, G, D, "cuda", layers=LAYERS)
    table, lens, logits, status = _prompt(be, m, cache, prompts, 96)
    assert int(status[1]) == 0
    histories = [list(p) for p in prompts]
    old = torch.zeros(B, 1)
    scores, parent, token = be.beam_select(logits[:, None], torch.zeros(B, 1, device="cuda"), W)
    for step in range(steps):
        # The chosen candidates' values, and that no better one was left out.  Both models round keys and values to
        # bf16; one that falls on the other side of a rounding moves its score by 2^-8 |q| |k| / sqrt(D) at most, and
        # with the weights here logits by less than 0.02.
        rows = len(histories) // B
        ref = torch.stack([plain.plain_logits(h) for h in histories]).view(B, rows, V)
        value = torch.log_softmax(ref, -1) + old.double().view(B, rows, 1)
        p, t = parent.cpu().long(), token.cpu().long()
        for b in range(B):
            mine = value[b, p[b] - b * rows, t[b]]
            assert float((mine - scores[b].cpu()).abs().max()) < 0.02
            best = torch.topk(value[b].flatten(), W).values
            assert float((best - mine.sort(descending=True).values).abs().max()) < 0.02
            assert len({(int(x), int(y)) for x, y in zip(p[b], t[b])}) == W
        histories = [histories[x] + [y] for x, y in zip(p.flatten().tolist(), t.flatten().tolist())]
        old = scores.cpu()
        table, lens, status = be.fork_pages(cache.pages, table, lens, parent.flatten(), 1)
        assert int(status[1]) == 0
        if step % 7 == 6:  # tidied up in between: nothing changes for the sequences
            table, _, live = be.compact_pages(cache.pages, table, lens + 1)
            assert int(table.max()) == int(live) - 1
        logits, lens = _step(be, m, cache, token.flatten(), table, lens)
        scores, parent, token = be.beam_select(logits.view(B, W, V), scores)
    assert lens.cpu().tolist() == [len(h) for h in histories]
    # Sequences end by having no child: with one left, only its pages are held.
    _, lens1, status = be.fork_pages(cache.pages, table, lens, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert int(status[0]) == 160 - -(-int(lens1) // PAGE)


def test_captured_decode_step(hip_backend):
    """A whole step -- preparation, attention, selection, fork -- in one graph, replayed with eager work
    between, against the same steps taken eagerly."""
    be, m, W, B = hip_backend, Model(8).cuda(), 4, 2
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5], [2, 7, 1]]

    def start():
        cache = PagedKVCache(100, PAGE, G, D, "cuda", layers=LAYERS)
        table, lens, logits, _ = _prompt(be, m, cache, prompts, 64)
        scores, parent, token = be.beam_select(logits[:, None], torch.zeros(B, 1, device="cuda"), W)
        table, lens, _ = be.fork_pages(cache.pages, table, lens, parent.flatten(), 1)
        return cache, [token.flatten(), scores, table, lens]

    def step(cache, state):
        token, scores, table, lens = state
        logits, lens = _step(be, m, cache, token, table, lens)
        scores, parent, token = be.beam_select(logits.view(B, W, V), scores)
        table, lens, status = be.fork_pages(cache.pages, table, lens, parent.flatten(), 1)
        return [token.flatten(), scores, table, lens], parent, status

    cache, state = start()
    want = []
    for _ in range(15):
        state, parent, status = step(cache, state)
        want.append([t.clone() for t in (*state, parent, status)])
    cache, state = start()
    step(cache, [t.clone() for t in state])  # warm up; it writes what the first step writes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, parent, status = step(cache, state)
        for a, b in zip(state, new):
            a.copy_(b)
    # Capturing runs nothing: the state is the start's.
    for i, w in enumerate(want):
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
            be.attention_paged(torch.randn(300, H, D, device="cuda"), *cache.layer(0),
                               state[2][:1].expand(300, -1).contiguous(), state[3][:1].expand(300).contiguous(), SCALE)
        got = [*state, parent, status]
        assert all(torch.equal(a, b) for a, b in zip(got, w)), i

"""The operators of a decode step over a paged KV cache, for timing.

``listed()`` names the workloads, ``draw(rng)`` gives further ones of the same
ranges, ``prepare`` makes what a serving program holds before the call, ``run``
is one pass through an operator -- in plain 32-bit torch operations, or, where
``own`` is true, through the public entry points of
``breezetoken_amd.backend.HipBackend`` -- ``work`` the bytes and operations a
pass cannot do without, ``exact`` the same results in 64 bits.

Kinds:

* ``attn``     one new token per sequence over a cache in pages;
* ``prep``     q/k norm, rotary positions and the writes of k and v into the
  pages, for a decode step's tokens or those of whole prompts;
* ``fork``     sequences continue their parents: shared pages, a copy of a
  shared last page that is written next, fresh pages for the tokens to come;
* ``compact``  live pages moved to the lowest places;
* ``beam``     the best continuations over beams and vocabulary.

A cache is ``pages`` (planes, N, page_size, Hkv * D) bf16, a plane for K and one
for V of each layer; ``table`` (rows, P) int32 holds each sequence's page ids
and ``lens`` (rows,) int32 its tokens.  What follows from a case alone (lengths,
parents) is drawn from the case's own ``shape`` number; ids and values come from
the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
THETA, EPS = 1.0e7, 1e-6

_shared: dict = {}


def _backend():
    """One backend per process, as a program holds it."""
    if "backend" not in _shared:
        from breezetoken_amd.backend import HipBackend

        _shared["backend"] = HipBackend(DEV)
    return _shared["backend"]


# ---------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # One chat's next token early on: a few hundred keys, launches and latency.
        dict(name="attn_chat", kind="attn", heads=8, kv_heads=2, dim=256, page=16, batch=1, shortest=301, longest=301,
             cap=4096, q="f32", out="f32", shape=1),
        # A small server's batch of similar lengths, head dimension 128, all bf16.
        dict(name="attn_batch", kind="attn", heads=32, kv_heads=8, dim=128, page=64, batch=24, shortest=1800,
             longest=3000, cap=4096, q="bf16", out="bf16", shape=2),
        # The benchmark's ragged batch, 256 to 32,768 tokens each.
        dict(name="attn_ragged", kind="attn", heads=8, kv_heads=2, dim=256, page=32, batch=32, shortest=256,
             longest=32768, cap=32768, q="f32", out="f32", shape=4),
        # The end of one very long context, 8 query heads per kv head.
        dict(name="attn_long", kind="attn", heads=16, kv_heads=2, dim=256, page=256, batch=1, shortest=131072,
             longest=131072, cap=131072, q="f32", out="f32", shape=5),
        # A decode step's 24 tokens: interleaved pairs over the whole head, no norm, no gate.
        dict(name="prep_step", kind="prep", heads=32, kv_heads=8, dim=128, page=64, rows=24, tokens=24, rope=128,
             inter=True, norm=False, gated=False, x="bf16", q="bf16", shape=6),
        # Five prompts of 8,192 tokens together: gated f32 projections, norm, a quarter of the head rotated.
        dict(name="prep_prompt", kind="prep", heads=8, kv_heads=2, dim=256, page=32, rows=5, tokens=8192, rope=64,
             inter=False, norm=True, gated=True, x="f32", q="f32", shape=7),
        # Four beams of one search take their parents' states; six layers' K and V.
        dict(name="fork_beams", kind="fork", planes=12, pages=320, page=16, width=512, rows=4, longest=1001, prefix=30,
             most=1, freed=0.0, shape=8),
        # A server's step: 128 sequences on common prefixes, some ended, some with a chunk of new tokens.
        dict(name="fork_server", kind="fork", planes=12, pages=2048, page=32, width=512, rows=128, longest=1500,
             prefix=16, most=64, freed=0.1, shape=9),
        # A small cache tidied up.
        dict(name="compact_small", kind="compact", planes=12, pages=300, page=16, width=512, rows=6, longest=700,
             prefix=7, shape=10),
        # A server's cache before long prompts are let in.
        dict(name="compact_server", kind="compact", planes=12, pages=2048, page=32, width=512, rows=64, longest=1500,
             prefix=16, shape=11),
        # One search of four beams over the benchmark model's vocabulary.
        dict(name="beam_one", kind="beam", batch=1, width=4, beams=4, vocab=248320, x="f32"),
        # A server's sixteen searches of eight beams each over the same vocabulary.
        dict(name="beam_server", kind="beam", batch=16, width=8, beams=8, vocab=248320, x="bf16"),
    ]


# (heads, kv heads, head dim): the 0.8B- and 35B-A3B-like attention layers and
# head dimensions 128 and 64 of other GQA models; group sizes 1 to 8.
SHAPES = ((8, 2, 256), (16, 2, 256), (32, 8, 128), (16, 2, 128), (15, 5, 64), (12, 12, 64), (7, 1, 128))
MOST_ATTN = 4.0e8  # bytes of keys and values of a drawn attention case


def _log(rng, lo: int, hi: int) -> int:
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng) -> dict:
    kind = rng.choice(("attn", "attn", "attn", "prep", "prep", "fork", "compact", "beam", "beam"))
    heads, kv_heads, dim = rng.choice(SHAPES)
    shape = rng.randrange(1 << 20)
    if kind == "attn":
        batch, longest = _log(rng, 1, 200), _log(rng, 1, 131072)
        while batch * longest * kv_heads * dim * 4 > MOST_ATTN:
            longest //= 2
        longest = max(1, longest)
        dtype = rng.choice(("f32", "bf16"))
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64, 128, 256)),
                    batch=batch, shortest=rng.choice((longest, max(1, longest // 2), max(1, longest // 100))),
                    longest=longest, cap=longest + rng.randrange(0, 2 * longest), q=dtype,
                    out=rng.choice(("f32", dtype)), shape=shape)
    if kind == "prep":
        rows = _log(rng, 1, 64)
        dtype = rng.choice(("f32", "bf16"))
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64, 128, 256)),
                    rows=rows, tokens=max(rows, _log(rng, 1, 6000)), rope=rng.choice((dim, dim // 2, dim // 4, 10)),
                    inter=rng.choice((True, False)), norm=rng.choice((True, False)), gated=rng.choice((True, False)),
                    x=dtype, q=rng.choice(("f32", dtype)), shape=shape)
    if kind in ("fork", "compact"):
        page, rows = rng.choice((16, 32, 64)), _log(rng, 1, 128)
        longest, prefix = _log(rng, 1, 1500), rng.choice((0, 1, 8))
        case = dict(kind=kind, planes=rng.choice((2, 8, 12)), page=page, width=rng.choice((128, 512, 640, 1024)),
                    rows=rows, longest=longest, prefix=prefix, shape=shape)
        # Free pages for a fresh one and `most` more tokens of each row, and a few.
        most = rng.choice((1, 1, 64))
        own_pages = rows * (-(-longest // page) - (-(-longest // page) > prefix) * min(prefix, longest // page))
        case["pages"] = prefix + own_pages + rows * (2 + most // page) + rng.randrange(1, 40)
        while case["planes"] > 2 and case["planes"] * case["pages"] * page * case["width"] * 2 > 6e8:
            case["planes"] -= 2
        while case["width"] > 128 and case["planes"] * case["pages"] * page * case["width"] * 2 > 6e8:
            case["width"] //= 2
        return dict(case, most=most, freed=rng.choice((0.0, 0.2))) if kind == "fork" else case
    width = _log(rng, 1, 16)
    vocab = _log(rng, 1000, 248320)
    batch = max(1, min(_log(rng, 1, 32), 16 * 8 * 248320 // (2 * width * vocab)))
    return dict(kind=kind, batch=batch, width=width, beams=rng.choice((width, width, 1, 2 * width, 13)), vocab=vocab,
                x=rng.choice(("f32", "bf16")))


# ------------------------------------------------------- what a case says itself
def _lengths(n: int, shortest: int, longest: int, rng) -> list[int]:
    """Log-uniform lengths, the last one the longest."""
    lo, hi = math.log(shortest), math.log(longest + 1)
    lens = [min(longest, int(math.exp(rng.uniform(lo, hi)))) for _ in range(n)]
    lens[-1] = longest
    return lens


def _plan(case: dict) -> dict:
    """Lengths, and for the page operators how rows share pages and which continue."""
    rng = random.Random(case["shape"])
    if case["kind"] == "attn":
        return dict(lens=_lengths(case["batch"], case["shortest"], case["longest"], rng))
    if case["kind"] == "prep":
        # Tokens dealt to rows; each row's run starts behind some cached tokens.
        rows, tokens = case["rows"], case["tokens"]
        cuts = sorted(rng.sample(range(1, tokens), rows - 1)) if rows > 1 else []
        runs = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
        return dict(runs=runs, first=[rng.randrange(0, 1500) for _ in runs])
    page, rows = case["page"], case["rows"]
    lens = _lengths(rows, max(1, case["longest"] // 3), case["longest"], rng)
    plan = dict(lens=lens, used=[-(-n // page) for n in lens],
                shared=[min(case["prefix"], n // page) for n in lens])
    if case["kind"] == "fork":
        plan["parent"] = [-1 if rng.random() < case["freed"] else rng.randrange(rows) for _ in range(rows)]
        plan["add"] = [rng.randint(0 if case["most"] > 1 else 1, case["most"]) for _ in range(rows)]
        plan["per_row"] = -(-(case["longest"] + case["most"]) // page)
    else:
        plan["per_row"] = -(-case["longest"] // page) + 2
    return plan


# --------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _dtype(name: str) -> torch.dtype:
    return torch.bfloat16 if name == "bf16" else torch.float32


def _randn(g: torch.Generator, *shape: int, dtype: str = "f32") -> torch.Tensor:
    return torch.randn(*shape, generator=g, device=DEV, dtype=_dtype(dtype))


def _int(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tables(cap: int, rope: int) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin (cap, rope) f32 from angles in 64 bits, both halves equal."""
    i = torch.arange(rope // 2, device=DEV, dtype=torch.float64)
    angle = torch.outer(torch.arange(cap, device=DEV, dtype=torch.float64), THETA ** (-2.0 * i / rope))
    angle = torch.cat((angle, angle), dim=1)
    return angle.cos().float(), angle.sin().float()


def prepare(case: dict, seed: int) -> dict:
    g, plan, kind = _gen(seed), None, case["kind"]
    state = dict(case=case)
    if kind == "beam":
        x = _randn(g, case["batch"], case["width"], case["vocab"]) * 3.0
        x[:, :, torch.randperm(case["vocab"], generator=g, device=DEV)[: case["vocab"] // 100]] = -math.inf  # barred tokens
        scores = -20.0 * torch.rand(case["batch"], case["width"], generator=g, device=DEV)
        return dict(state, logits=x.to(_dtype(case["x"])), scores=scores)
    plan = _plan(case)
    if kind in ("fork", "compact"):
        N, page, rows, width = case["pages"], case["page"], case["rows"], plan["per_row"]
        ids = torch.randperm(N, generator=g, device=DEV).to(torch.int32).cpu().numpy()
        table = np.full((rows, width), -1, dtype=np.int32)
        at = case["prefix"]
        for i, (n, shared) in enumerate(zip(plan["used"], plan["shared"])):
            table[i, :shared] = ids[:shared]
            table[i, shared:n] = ids[at : at + n - shared]
            at += n - shared
        pages = _randn(g, case["planes"], N, page, case["width"], dtype="bf16")
        state.update(pages=pages, table=_int(table), lens=_int(plan["lens"]))
        if kind == "fork":
            state.update(parent=_int(plan["parent"]), add=_int(plan["add"]))
        return state
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if kind == "attn":
        lens, per_row = plan["lens"], -(-case["cap"] // page)
    else:
        lens = [a + n for a, n in zip(plan["first"], plan["runs"])]
        per_row = -(-max(lens) // page)
    used = [-(-n // page) for n in lens]
    N = sum(used) + max(1, sum(used) // 8)
    ids = torch.randperm(N, generator=g, device=DEV).to(torch.int32).cpu().numpy()
    table = np.full((len(lens), per_row), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = ids[at : at + n]
        at += n
    k = _randn(g, N, page, G, D, dtype="bf16")
    v = _randn(g, N, page, G, D, dtype="bf16")
    state.update(k=k, v=v, table=_int(table))
    if kind == "attn":
        return dict(state, q=_randn(g, case["batch"], H, D, dtype=case["q"]), lens=_int(lens))
    qkv = _randn(g, case["tokens"], (2 if case["gated"] else 1) * H * D + 2 * G * D, dtype=case["x"])
    cos, sin = _tables(max(lens), case["rope"])
    rows = np.repeat(np.arange(len(lens)), plan["runs"])
    pos = np.concatenate([a + np.arange(n) for a, n in zip(plan["first"], plan["runs"])])
    norm = (1.0 + 0.1 * _randn(g, D), 1.0 + 0.1 * _randn(g, D)) if case["norm"] else (None, None)
    return dict(state, qkv=qkv, cos=cos, sin=sin, rows=_int(rows), pos=_int(pos), norm=norm)


# ------------------------------------------------------------------ plain forms
def _plain_attn(s: dict) -> torch.Tensor:
    q, lens, table, k, v = s["q"], s["lens"], s["table"], s["k"], s["v"]
    B, H, D = q.shape
    N, page, G, _ = k.shape
    n = -(-s["case"]["longest"] // page)  # the program knows its longest sequence
    ids = table[:, :n].clamp(min=0).long()
    keys = k[ids].reshape(B, n * page, G, D).permute(0, 2, 3, 1).float().contiguous()
    x = torch.matmul(q.float().view(B, G, H // G, D), keys) * D**-0.5
    del keys
    live = torch.arange(n * page, device=q.device) < lens[:, None]
    x = x.masked_fill(~live[:, None, None, :], -math.inf)
    x = torch.exp(x - x.amax(dim=-1, keepdim=True))
    x = x / x.sum(dim=-1, keepdim=True)
    values = v[ids].reshape(B, n * page, G, D).permute(0, 2, 1, 3).float().contiguous()
    return torch.matmul(x, values).reshape(B, H, D).to(_dtype(s["case"]["out"]))


def _plain_turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, rope: int, inter: bool) -> torch.Tensor:
    """x (T, heads, D) with its first ``rope`` values rotated; cos / sin (T, 1, rope / 2)."""
    head, rest = x[..., :rope], x[..., rope:]
    a, b = (head[..., 0::2], head[..., 1::2]) if inter else (head[..., : rope // 2], head[..., rope // 2 :])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((a, b), dim=-1).flatten(-2) if inter else torch.cat((a, b), dim=-1)
    return torch.cat((head, rest), dim=-1)


def _plain_norm(x: torch.Tensor, w: torch.Tensor | None) -> torch.Tensor:
    return x if w is None else x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w


def _plain_prep(s: dict) -> dict:
    case, qkv, k, v = s["case"], s["qkv"], s["k"], s["v"]
    H, G, D, rope = case["heads"], case["kv_heads"], case["dim"], case["rope"]
    T, page, nq = qkv.shape[0], k.shape[1], (2 if case["gated"] else 1) * H * D
    x = qkv.float()
    q = x[:, :nq].view(T, H, -1)[..., :D]
    new_k, new_v = x[:, nq : nq + G * D].view(T, G, D), x[:, nq + G * D :].view(T, G, D)
    at = s["pos"].long()
    cos, sin = s["cos"][at][:, None, : rope // 2], s["sin"][at][:, None, : rope // 2]
    q = _plain_turn(_plain_norm(q, s["norm"][0]), cos, sin, rope, case["inter"])
    new_k = _plain_turn(_plain_norm(new_k, s["norm"][1]), cos, sin, rope, case["inter"])
    slot = s["table"][s["rows"].long(), at // page].long() * page + at % page
    k.view(-1, G, D)[slot] = new_k.to(k.dtype)
    v.view(-1, G, D)[slot] = new_v.to(v.dtype)
    return dict(q=q.to(_dtype(case["q"])), k=k, v=v)


def _plain_fork(s: dict) -> dict:
    pages, table, page = s["pages"], s["table"], s["case"]["page"]
    planes, N, _, width = pages.shape
    P = table.shape[1]
    keep = (s["parent"] >= 0)[:, None]
    parent = s["parent"].clamp(min=0).long()
    lens = torch.where(keep[:, 0], s["lens"][parent], 0)
    column = torch.arange(P, device=table.device)
    used = (lens + page - 1) // page
    new = torch.where(keep & (column < used[:, None]), table[parent], -1)
    held = torch.zeros(N + 1, dtype=torch.int32, device=table.device)
    held.scatter_add_(0, torch.where(new < 0, N, new).flatten().long(), torch.ones_like(new).flatten())
    # A shared, partly filled last page that will be written is replaced by a fresh one.
    last = new.gather(1, (used - 1).clamp(min=0)[:, None].long())[:, 0]
    fork = (s["add"] > 0) & (lens % page > 0) & (held[last.clamp(min=0).long()] > 1)
    need = (lens + s["add"] + page - 1) // page
    fresh = (column >= used[:, None]) & (column < need[:, None]) | (column == used[:, None] - 1) & fork[:, None]
    order = torch.argsort((held[:N] > 0).to(torch.int8), stable=True).to(torch.int32)  # free pages, lowest first
    rank = torch.cumsum(fresh.flatten(), 0).view_as(new) - 1
    new = torch.where(fresh, order[rank.clamp(min=0)], new)
    at = fork.nonzero()[:, 0]
    source, target = last[at].long(), new[at, (used[at] - 1).long()].long()
    token = torch.arange(page, device=table.device)
    some = (token < (lens[at] % page)[:, None]).flatten().nonzero()[:, 0]
    source, target = (source[:, None] * page + token).flatten()[some], (target[:, None] * page + token).flatten()[some]
    flat = pages.view(planes, N * page, width)
    flat[:, target] = flat[:, source]
    left = (held[:N] == 0).sum() - fresh.sum()
    return dict(table=new, lens=lens, status=torch.stack((left, torch.zeros_like(left))).to(torch.int32), pages=pages)


def _plain_compact(s: dict) -> dict:
    pages, table, page = s["pages"], s["table"], s["case"]["page"]
    N, P = pages.shape[1], table.shape[1]
    used = torch.arange(P, device=table.device) < ((s["lens"] + page - 1) // page)[:, None]
    held = torch.zeros(N + 1, dtype=torch.bool, device=table.device)
    held[torch.where(used, table, N).flatten().long()] = True
    held = held[:N]
    live = held.sum()
    index = torch.arange(N, device=table.device)
    source, target = (held & (index >= live)).nonzero()[:, 0], (~held & (index < live)).nonzero()[:, 0]
    where = torch.where(held, index, -1)
    where[source] = target
    pages[:, target] = pages[:, source]
    new = torch.where(used, where[table.clamp(min=0).long()], -1)
    return dict(table=new.to(torch.int32), where=where.to(torch.int32), live=live.to(torch.int32).view(1), pages=pages)


def _plain_beam(s: dict) -> dict:
    # In 64 bits: candidates of two beams can lie nearer to each other than 32 bits resolve.
    x = s["logits"].double()
    B, W, V = x.shape
    top = x.amax(dim=-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))) + s["scores"].double()[..., None]
    x, at = torch.sort(x.view(B, W * V), dim=1, descending=True, stable=True)
    at = at[:, : s["case"]["beams"]]
    parent = at // V + torch.arange(B, device=at.device)[:, None] * W
    return dict(scores=x[:, : s["case"]["beams"]].float(), parent=parent.to(torch.int32), token=(at % V).to(torch.int32))


# --------------------------------------------------------------------- one pass
def _own(s: dict):
    case, be = s["case"], _backend()
    kind = case["kind"]
    if kind == "attn":
        return be.attention_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], case["dim"] ** -0.5,
                                  out_dtype=_dtype(case["out"]))
    if kind == "prep":
        q, _ = be.attn_prep_paged(s["qkv"], s["norm"][0], s["norm"][1], EPS, s["cos"], s["sin"], s["pos"], case["rope"],
                                  s["k"], s["v"], s["table"], case["heads"], case["kv_heads"], case["dim"],
                                  rows=s["rows"], gated=case["gated"], interleaved=case["inter"],
                                  q_dtype=_dtype(case["q"]))
        return dict(q=q, k=s["k"], v=s["v"])
    if kind == "fork":
        table, lens, status = be.fork_pages(s["pages"], s["table"], s["lens"], s["parent"], s["add"])
        return dict(table=table, lens=lens, status=status, pages=s["pages"])
    if kind == "compact":
        table, where, live = be.compact_pages(s["pages"], s["table"], s["lens"])
        return dict(table=table, where=where, live=live, pages=s["pages"])
    scores, parent, token = be.beam_select(s["logits"], s["scores"], case["beams"])
    return dict(scores=scores, parent=parent, token=token)


_PLAIN = dict(attn=_plain_attn, prep=_plain_prep, fork=_plain_fork, compact=_plain_compact, beam=_plain_beam)


def run(state: dict):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "beam":
        n = case["batch"] * case["width"] * case["vocab"]
        return dict(bytes=n * (2 if case["x"] == "bf16" else 4) + case["batch"] * (4 * case["width"] + 12 * case["beams"]),
                    flops=4 * n)
    plan, page = _plan(case), case["page"]
    if kind in ("fork", "compact"):
        rows, token = case["rows"], case["planes"] * case["width"] * 2
        cells = 4 * (sum(plan["used"]) + 2 * rows + rows * plan["per_row"])
        if kind == "compact":
            # Where the live pages lie is drawn from the seed: those past their count move.
            live = min(case["prefix"], max(plan["shared"])) + sum(n - m for n, m in zip(plan["used"], plan["shared"]))
            return dict(bytes=cells + 4 * case["pages"] + 2 * live * (1 - live / case["pages"]) * page * token, flops=0)
        count: dict = {}
        for a in plan["parent"]:
            if a >= 0:
                j = plan["used"][a] - 1
                key = j if j < plan["shared"][a] else (a, j)
                count[key] = count.get(key, 0) + 1
        tokens = 0
        for a, add in zip(plan["parent"], plan["add"]):
            if a >= 0 and add > 0 and plan["lens"][a] % page and count[(a, plan["used"][a] - 1)] > 1:
                tokens += plan["lens"][a] % page
        return dict(bytes=cells + 2 * tokens * token, flops=0)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if kind == "attn":
        tokens = sum(plan["lens"])
        rows = case["batch"] * H * D
        entries = sum(-(-n // page) for n in plan["lens"])
        return dict(bytes=tokens * G * D * 4 + rows * ((2 if case["q"] == "bf16" else 4) + (2 if case["out"] == "bf16" else 4))
                    + 4 * (entries + case["batch"]), flops=4 * tokens * H * D)
    T, size = case["tokens"], 2 if case["x"] == "bf16" else 4
    positions = len({p for a, n in zip(plan["first"], plan["runs"]) for p in range(a, a + n)})
    return dict(bytes=T * (H + 2 * G) * D * size + T * H * D * (2 if case["q"] == "bf16" else 4) + T * G * D * 4
                + positions * case["rope"] * 4 + 8 * T, flops=T * (H + G) * (3 * case["rope"] + (4 * D if case["norm"] else 0)))


# ---------------------------------------------------------------- 64-bit results
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return dict(attn=_exact_attn, prep=_exact_prep, fork=_exact_fork, compact=_exact_compact, beam=_exact_beam)[case["kind"]](s)


def _exact_attn(s: dict) -> torch.Tensor:
    q, k, v = s["q"].double(), s["k"], s["v"]
    B, H, D = q.shape
    page, G = k.shape[1], k.shape[2]
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["table"][b, : -(-n // page)].long()
        keys, values = k[ids].reshape(-1, G, D)[:n], v[ids].reshape(-1, G, D)[:n]
        for h in range(H):
            x = (keys[:, h // (H // G)].double() * q[b, h]).sum(dim=1) / math.sqrt(D)
            p = torch.softmax(x, dim=0)
            out[b, h] = (values[:, h // (H // G)].double() * p[:, None]).sum(dim=0)
    return out


def _exact_prep(s: dict) -> dict:
    case, k, v = s["case"], s["k"].double(), s["v"].double()
    H, G, D, rope, page = case["heads"], case["kv_heads"], case["dim"], case["rope"], case["page"]
    T = case["tokens"]
    half = rope // 2
    x = s["qkv"].double()
    step = 2 * D if case["gated"] else D
    columns = torch.arange(H * step, device=x.device).view(H, step)[:, :D].reshape(-1)
    q = x[:, columns].reshape(T, H, D)
    base = H * step
    new_k = x[:, base : base + G * D].reshape(T, G, D)
    new_v = x[:, base + G * D : base + 2 * G * D].reshape(T, G, D)
    pos = s["pos"].long()
    if case["norm"]:
        q = q / torch.sqrt(q.square().sum(-1, keepdim=True) / D + EPS) * s["norm"][0].double()
        new_k = new_k / torch.sqrt(new_k.square().sum(-1, keepdim=True) / D + EPS) * s["norm"][1].double()
    # As a complex product: value i turned by the angle of column i.
    turn = torch.complex(s["cos"][pos][:, :half].double(), s["sin"][pos][:, :half].double())[:, None]
    first = torch.arange(half, device=x.device) * (2 if case["inter"] else 1)
    second = first + (1 if case["inter"] else half)
    for t in (q, new_k):
        z = torch.complex(t[..., first].contiguous(), t[..., second].contiguous()) * turn
        t[..., first], t[..., second] = z.real, z.imag
    row, col = s["rows"].long(), torch.div(pos, page, rounding_mode="floor")
    ids = s["table"][row, col].long()
    k[ids, pos - col * page] = new_k
    v[ids, pos - col * page] = new_v
    return dict(q=q, k=k, v=v)


def _exact_fork(s: dict) -> dict:
    pages, page = s["pages"].clone(), s["case"]["page"]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    N, P = pages.shape[1], len(table[0])
    new, new_lens, holders = [], [], {}
    for p in s["parent"].tolist():
        n = lens[p] if p >= 0 else 0
        row = table[p][: -(-n // page)] if n else []
        new.append(list(row))
        new_lens.append(n)
        for i in row:
            holders[i] = holders.get(i, 0) + 1
    free = [i for i in range(N) if i not in holders]
    for row, n, add in zip(new, new_lens, s["add"].tolist()):
        if add and n % page and holders[row[-1]] > 1:
            target = free.pop(0)
            pages[:, target, : n % page] = s["pages"][:, row[-1], : n % page]
            row[-1] = target
        while len(row) < -(-(n + add) // page):
            row.append(free.pop(0))
    new = [row + [-1] * (P - len(row)) for row in new]
    return dict(table=_int(new), lens=_int(new_lens), status=_int([len(free), 0]), pages=pages)


def _exact_compact(s: dict) -> dict:
    pages, page = s["pages"].clone(), s["case"]["page"]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    N, P = pages.shape[1], len(table[0])
    rows = [row[: -(-n // page)] for row, n in zip(table, lens)]
    live = sorted({i for row in rows for i in row})
    holes = sorted(set(range(len(live))) - set(live))
    where = {i: i for i in live}
    for i in [i for i in live if i >= len(live)]:
        where[i] = holes.pop(0)
        pages[:, where[i]] = s["pages"][:, i]
    new = [[where[i] for i in row] + [-1] * (P - len(row)) for row in rows]
    return dict(table=_int(new), where=_int([where.get(i, -1) for i in range(N)]), live=_int([len(live)]), pages=pages)


def _exact_beam(s: dict) -> dict:
    out = dict(scores=[], parent=[], token=[])
    B, W, V = s["logits"].shape
    K = s["case"]["beams"]
    for b in range(B):
        found = []
        for w in range(W):
            x = s["logits"][b, w].double()
            x = torch.log_softmax(x, dim=0) + float(s["scores"][b, w])
            least = float(torch.topk(x, min(K, V)).values[-1])
            at = (x >= least).nonzero()[:, 0]
            found += [(-p, w, t) for p, t in zip(x[at].tolist(), at.tolist())]
        found = sorted(found)[:K]
        out["scores"].append([-p for p, _, _ in found])
        out["parent"].append([b * W + w for _, w, _ in found])
        out["token"].append([t for _, _, t in found])
    return dict(scores=torch.tensor(out["scores"], dtype=torch.float64, device=DEV), parent=_int(out["parent"]),
                token=_int(out["token"]))

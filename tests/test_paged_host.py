"""What the paged cache's operators refuse, at both interfaces, without a GPU:
nothing is launched (the C entry points return before, the Python ones raise before)."""

from __future__ import annotations

import math

import pytest
import torch

from breezetoken_amd import PagedKVCache, _lib
from breezetoken_amd.backend import HipBackend, rope_tables, rope_tables_scaled

A = 1 << 20  # an aligned address that no refused call touches


class _NoLaunch(HipBackend):
    """The argument checks of HipBackend over host tensors; a launch fails the test."""

    def __init__(self):
        self._dev = torch.device("cpu")
        self._lib = _lib.lib()

    def _run(self, name, *args):
        raise AssertionError(f"{name} was launched")


@pytest.fixture
def be():
    return _NoLaunch()


# ------------------------------------------------------------------ C interface
ATTN = dict(q=A, q_dtype=0, q_stride=8 * 128, k=A, v=A, sp=16 * 256, st=256, sh=128, pages=4, page=16, table=A, ts=4,
            per_seq=4, lens=A, batch=1, heads=8, kv_heads=2, dim=128, scale=1.0, ws=A, ws_bytes=1 << 40, out=A, out_dtype=0,
            out_stride=8 * 128, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -22), (dict(k=None), -22), (dict(v=None), -22), (dict(table=None), -22), (dict(lens=None), -22),
    (dict(out=None), -22), (dict(q=A + 8), -22), (dict(k=A + 2), -22), (dict(table=A + 2), -22), (dict(q_dtype=2), -22),
    (dict(out_dtype=-1), -22), (dict(q_stride=1016), -22), (dict(q_stride=1028), -22), (dict(out_stride=8), -22),
    (dict(sp=0), -22), (dict(st=4), -22), (dict(sh=-128), -22), (dict(st=250), -22), (dict(pages=0), -22),
    (dict(per_seq=0), -22), (dict(ts=3), -22), (dict(batch=0), -22), (dict(heads=9), -22), (dict(kv_heads=0), -22),
    (dict(page=8), -95), (dict(page=48), -95), (dict(page=2048), -95), (dict(dim=96, q_stride=1024), -95),
    (dict(heads=18, q_stride=4096, out_stride=4096), -95), (dict(batch=4097), -95),
    (dict(batch=4096, heads=2048, kv_heads=2048, q_stride=1 << 18, out_stride=1 << 18), -95),
    (dict(per_seq=1 << 28, ts=1 << 28), -95), (dict(st=1 << 28), -95),
])
def test_attention_refuses(change, code):
    assert _lib.lib().bt_gqa_decode_paged(*{**ATTN, **change}.values()) == code


PREP = dict(qkv=A, dtype=0, stride=2 * 8 * 128 + 512, tokens=3, heads=8, kv_heads=2, dim=128, gated=1, qn=A, kn=A, eps=1e-6,
            cos=A, sin=A, rope=64, cap=10, inter=0, pos=A, rows=None, q=A, q_dtype=0, k=A, v=A, sp=16 * 256, st=256, sh=128,
            pages=4, page=16, table=A, ts=4, table_rows=3, per_seq=4, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(qkv=None), -22), (dict(pos=None), -22), (dict(q=None), -22), (dict(k=None), -22), (dict(table=None), -22),
    (dict(qkv=A + 4), -22), (dict(q=A + 4), -22), (dict(dtype=7), -22), (dict(q_dtype=7), -22), (dict(stride=2552), -22),
    (dict(stride=2564), -22), (dict(tokens=0), -22), (dict(heads=0), -22), (dict(table_rows=0), -22), (dict(kn=None), -22),
    (dict(sin=None), -22), (dict(qn=A + 4), -22), (dict(rope=0), -22), (dict(rope=63), -22), (dict(rope=130), -22),
    (dict(cap=0), -22), (dict(eps=-1.0), -22), (dict(eps=math.nan), -22), (dict(sh=0), -22), (dict(ts=1), -22),
    (dict(page=12), -95), (dict(dim=96), -95), (dict(tokens=1 << 30), -95),
])
def test_prep_refuses(change, code):
    assert _lib.lib().bt_attn_prep_paged(*{**PREP, **change}.values()) == code


FORK = dict(pages=A, plane=64 * 1024, stride=1024, planes=2, num=64, page=16, elems=64, table=A, lens=A, rows=3, per_seq=4,
            parent=A, add=A, rows_out=5, keep=None, num_keep=0, table_out=2 * A, lens_out=2 * A, status=A, ws=A,
            ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(pages=None), -22), (dict(pages=A + 2), -22), (dict(plane=1000), -22), (dict(stride=1016), -22), (dict(planes=0), -22),
    (dict(num=0), -22), (dict(elems=4), -22), (dict(elems=60), -22), (dict(table=None), -22), (dict(lens=None), -22),
    (dict(rows=-1), -22), (dict(rows_out=-1), -22), (dict(per_seq=0), -22), (dict(parent=None), -22), (dict(num_keep=2), -22),
    (dict(table_out=None), -22), (dict(table_out=A), -22), (dict(lens_out=None), -22), (dict(lens_out=A), -22),
    (dict(status=None), -22), (dict(plane=2048), -22), (dict(page=24), -95), (dict(per_seq=1 << 30), -95),
    (dict(planes=8192, plane=1 << 20, stride=1024, num=1024), -95),
    (dict(ws=None), -28), (dict(ws_bytes=64), -28), (dict(ws=A + 4), -28),
])
def test_fork_refuses(change, code):
    assert _lib.lib().bt_fork_pages(*{**FORK, **change}.values()) == code


COMPACT = dict(pages=A, plane=64 * 1024, stride=1024, planes=2, num=64, page=16, elems=64, table=A, lens=A, rows=3, per_seq=4,
               keep=None, num_keep=0, table_out=2 * A, where=A, live=A, ws=A, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(pages=None), -22), (dict(where=None), -22), (dict(live=None), -22), (dict(table_out=A), -22), (dict(page=100), -95),
    (dict(num_keep=-1), -22), (dict(ws_bytes=0), -28),
])
def test_compact_refuses(change, code):
    assert _lib.lib().bt_compact_pages(*{**COMPACT, **change}.values()) == code


BEAM = dict(logits=A, dtype=0, sb=400, sw=100, scores=A, batch=2, width=4, vocab=100, beams=4, so=A, po=A, to=A, ws=A,
            ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), -22), (dict(scores=None), -22), (dict(so=None), -22), (dict(po=None), -22), (dict(to=None), -22),
    (dict(dtype=3), -22), (dict(sb=-1), -22), (dict(sw=-100), -22), (dict(batch=0), -22), (dict(width=0), -22),
    (dict(vocab=0), -22), (dict(beams=0), -22), (dict(vocab=1, beams=5), -22), (dict(logits=A + 2), -22), (dict(width=65), -95),
    (dict(beams=65), -95), (dict(batch=1 << 30), -95), (dict(batch=1 << 19), -95), (dict(ws=None), -28), (dict(ws_bytes=8), -28),
])
def test_beam_refuses(change, code):
    assert _lib.lib().bt_beam_select(*{**BEAM, **change}.values()) == code


def test_workspace_sizes_refuse_malformed_shapes():
    lib = _lib.lib()
    assert lib.bt_paged_workspace_bytes(0, 8, 2, 128, 64) == 0 and lib.bt_paged_workspace_bytes(1, 8, 3, 128, 64) == 0
    assert lib.bt_pages_workspace_bytes(0, 4) == 0 and lib.bt_pages_workspace_bytes(4, -1) == 0
    assert lib.bt_beam_workspace_bytes(1, 0, 4, 4) == 0
    assert lib.bt_pages_workspace_bytes(100, 7) > 0 and lib.bt_beam_workspace_bytes(1, 4, 100, 4) > 0


# ------------------------------------------------------------- Python interface
def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def _attn(**kw):
    a = dict(q=torch.zeros(2, 8, 128), k=_bf(4, 16, 2, 128), v=_bf(4, 16, 2, 128), table=torch.zeros(2, 3, dtype=torch.int32),
             lens=_i(1, 2), scale=1.0)
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(8, 128)), dict(q=torch.zeros(2, 8, 64)), dict(q=torch.zeros(2, 7, 128)), dict(q=torch.zeros(2, 0, 128)),
    dict(q=torch.zeros(2, 18, 128)), dict(q=torch.zeros(2, 8, 128, dtype=torch.float16)),
    dict(q=torch.zeros(2, 8, 128).double()), dict(k=torch.zeros(4, 16, 2, 128)), dict(v=_bf(4, 16, 1, 128)),
    dict(k=_bf(4, 24, 2, 128), v=_bf(4, 24, 2, 128)), dict(k=_bf(4, 8, 2, 128), v=_bf(4, 8, 2, 128)),
    dict(k=_bf(0, 16, 2, 128), v=_bf(0, 16, 2, 128)), dict(k=_bf(4, 2, 16, 128).transpose(1, 2)),
    dict(k=_bf(4, 16, 128, 2).transpose(2, 3), v=_bf(4, 16, 128, 2).transpose(2, 3)),
    dict(table=torch.zeros(2, 3, dtype=torch.int64)), dict(table=torch.zeros(3, 3, dtype=torch.int32)),
    dict(table=torch.zeros(3, 2, dtype=torch.int32).t()), dict(table=torch.zeros(2, 0, dtype=torch.int32)),
    dict(table=_i(1, 2)), dict(lens=_i(1)), dict(lens=torch.tensor([1, 2])), dict(lens=_i(1, 2, 3, 4)[::2]),
    dict(lens=_i(1, 2).to("meta")), dict(out_dtype=torch.float16), dict(q=torch.zeros(2, 8, 96), k=_bf(4, 16, 2, 96), v=_bf(4, 16, 2, 96)),
])
def test_attention_paged_raises(be, kw):
    with pytest.raises(RuntimeError):
        be.attention_paged(**_attn(**kw))


def _prep(**kw):
    a = dict(qkv=torch.zeros(2, 2 * 4 * 64 + 2 * 2 * 64), q_norm=torch.ones(64), k_norm=torch.ones(64), eps=1e-6,
             cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), pos=_i(0, 1), rope_dim=32, k=_bf(4, 16, 2, 64), v=_bf(4, 16, 2, 64),
             table=torch.zeros(2, 3, dtype=torch.int32), heads=4, kv_heads=2, head_dim=64)
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(qkv=torch.zeros(2, 100)), dict(qkv=torch.zeros(768)), dict(qkv=torch.zeros(2, 768, dtype=torch.float16)),
    dict(gated=False), dict(head_dim=96), dict(heads=3), dict(kv_heads=0), dict(q_norm=None), dict(k_norm=None), dict(cos=None),
    dict(sin=torch.zeros(8, 32)), dict(cos=torch.zeros(9, 32).double(), sin=torch.zeros(9, 32).double()),
    dict(cos=torch.zeros(9, 30), sin=torch.zeros(9, 30)), dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)),
    dict(cos=torch.zeros(32, 9).t(), sin=torch.zeros(32, 9).t()), dict(q_norm=torch.ones(64).double()),
    dict(q_norm=torch.ones(32), k_norm=torch.ones(64)), dict(rope_dim=31), dict(rope_dim=0), dict(rope_dim=66),
    dict(pos=_i(0)), dict(pos=torch.tensor([0, 1])), dict(rows=_i(0)), dict(rows=torch.tensor([0, 1])),
    dict(table=torch.zeros(1, 3, dtype=torch.int32)), dict(k=_bf(4, 16, 1, 64), v=_bf(4, 16, 1, 64)),
    dict(k=_bf(4, 16, 2, 128), v=_bf(4, 16, 2, 128)), dict(q_dtype=torch.float16), dict(table=torch.zeros(2, 3).int().to("meta")),
])
def test_attn_prep_paged_raises(be, kw):
    with pytest.raises((RuntimeError, ValueError)):
        be.attn_prep_paged(**_prep(**kw))


def _fork(**kw):
    a = dict(pages=_bf(2, 6, 16, 64), table=torch.zeros(3, 4, dtype=torch.int32), lens=_i(1, 2, 3))
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(pages=torch.zeros(2, 6, 16, 64)), dict(pages=_bf(6, 16, 64)), dict(pages=_bf(2, 0, 16, 64)), dict(pages=_bf(2, 6, 24, 64)),
    dict(pages=_bf(2, 6, 16, 60)), dict(pages=_bf(2, 6, 64, 16).transpose(2, 3)), dict(pages=_bf(2, 6, 16, 128)[..., :64]),
    dict(table=torch.zeros(3, 4)), dict(table=torch.zeros(4, 3, dtype=torch.int32).t()), dict(lens=_i(1)),
    dict(lens=torch.tensor([1, 2, 3])), dict(keep=torch.tensor([1])), dict(keep=_i(1).to("meta")),
])
def test_page_operators_raise(be, kw):
    for op in (be.fork_pages, be.compact_pages):
        with pytest.raises(RuntimeError):
            op(**_fork(**kw))


@pytest.mark.parametrize("kw", [dict(parent=torch.tensor([1])), dict(parent=_i(1, 2), add=_i(1)), dict(add=torch.tensor([1, 1, 1])),
                                dict(add=-1), dict(add=1 << 31), dict(add=1.5), dict(parent=_i(0).to("meta"))])
def test_fork_raises(be, kw):
    with pytest.raises((RuntimeError, ValueError, TypeError)):
        be.fork_pages(**_fork(**kw))


@pytest.mark.parametrize("logits,scores,beams", [
    (torch.zeros(2, 9), torch.zeros(2), 1), (torch.zeros(2, 3, 9), torch.zeros(2, 2), 1), (torch.zeros(2, 3, 0), torch.zeros(2, 3), 1),
    (torch.zeros(2, 0, 9), torch.zeros(2, 0), 1), (torch.zeros(2, 3, 9), torch.zeros(2, 3), 0),
    (torch.zeros(2, 3, 1), torch.zeros(2, 3), 4), (torch.zeros(1, 65, 9), torch.zeros(1, 65), 1),
    (torch.zeros(1, 3, 99), torch.zeros(1, 3), 65), (torch.zeros(2, 3, 9).half(), torch.zeros(2, 3), 1),
    (torch.zeros(2, 3, 9), torch.zeros(2, 3).double(), 1), (torch.zeros(2, 3, 9).to("meta"), torch.zeros(2, 3), 1),
])
def test_beam_select_raises(be, logits, scores, beams):
    with pytest.raises((RuntimeError, ValueError)):
        be.beam_select(logits, scores, beams)


# ---------------------------------------------------------------- cache, tables
def test_paged_cache_views():
    c = PagedKVCache(6, 16, 2, 64, "cpu", layers=3)
    assert c.pages.shape == (6, 6, 16, 128) and c.nbytes() == 6 * 6 * 16 * 128 * 2
    k, v = c.layer(1)
    k[2, 3, 1, 5], v[5, 15, 0, 0] = 1.0, 2.0
    assert float(c.pages[2, 2, 3, 64 + 5]) == 1.0 and float(c.pages[3, 5, 15, 0]) == 2.0
    rk, rv = c.rows(1, 2, 20)
    assert rk.shape == (20, 2, 64) and float(rk[3, 1, 5]) == 1.0 and rk.data_ptr() == k[2].data_ptr()
    table, lens = c.empty_table(4, 33)
    assert table.shape == (4, 3) and bool((table == -1).all()) and lens.tolist() == [0] * 4
    for bad in (lambda: c.layer(3), lambda: c.layer(-1), lambda: c.rows(0, 5, 17), lambda: c.rows(0, -1, 1)):
        with pytest.raises(IndexError):
            bad()
    for args in ((0, 16, 2, 64), (4, 17, 2, 64), (4, 16, 0, 64), (4, 16, 1, 4), (4, 16, 2, 64, "cpu", 0)):
        with pytest.raises(ValueError):
            PagedKVCache(*args, *(() if len(args) > 4 else ("cpu",)))
    with pytest.raises(ValueError):
        c.empty_table(1, 0)


def test_scaled_tables():
    plain = rope_tables(300, 64, 1.0e4, "cpu")
    for method, trained in (("linear", None), ("ntk", None), ("yarn", 4096)):
        cos, sin = rope_tables_scaled(300, 64, 1.0e4, method, 1.0, trained, "cpu")
        # f32 angles of up to 300 are off by a few half steps of 300.
        assert float((cos - plain[0]).abs().max()) <= 300 * 4 * 2.0**-24
        assert torch.equal(cos[:, :32], cos[:, 32:]) and cos.dtype == torch.float32
    # linear: position 8 p at factor 8 has position p's angles; ntk: the first pair keeps its rate, the last is
    # slowed by the factor; yarn: likewise, times the attention factor.
    base = rope_tables_scaled(64, 64, 1.0e4, "linear", 1.0, device="cpu")
    lin = rope_tables_scaled(512, 64, 1.0e4, "linear", 8.0, device="cpu")
    assert float((lin[1][::8] - base[1]).abs().max()) <= 2.0**-22
    ntk = rope_tables_scaled(512, 64, 1.0e4, "ntk", 8.0, device="cpu")
    assert float((ntk[1][:64, 0] - base[1][:, 0]).abs().max()) <= 2.0**-22
    assert float((ntk[1][::8, 31] - base[1][:, 31]).abs().max()) <= 2.0**-22
    yarn = rope_tables_scaled(512, 64, 1.0e4, "yarn", 8.0, 4096, "cpu")
    factor = 0.1 * math.log(8.0) + 1.0
    assert float((yarn[1][:64, 0] / factor - base[1][:, 0]).abs().max()) <= 2.0**-22
    assert float((yarn[1][::8, 31] / factor - base[1][:, 31]).abs().max()) <= 2.0**-22
    for bad in (("yarn", 8.0), ("other", 8.0), ("linear", 0.5)):
        with pytest.raises(ValueError):
            rope_tables_scaled(16, 64, 1.0e4, *bad, device="cpu")
    with pytest.raises(ValueError):
        rope_tables_scaled(16, 63, 1.0e4, "linear", 2.0, device="cpu")

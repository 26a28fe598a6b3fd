"""Refusals of attention over windows and of trees and of rows that turn by given positions: what the host can
see is checked before anything is launched (no GPU, the pointers are never read)."""
import ctypes as C
import math
import random

import pytest

from test_paged import BAD_BATCH, BAD_KV, EINVAL, P, batch, kv


def window(qa, kvd={}, bd={}, **k):
    d = dict(out=P, q=P + 4096, dtype=qa.ST_F32, heads=4, scale=0.1, window=100, sinks=4, ws=P, ws_bytes=1 << 40)
    d.update(k)
    a, b = kv(qa, **kvd), batch(qa, **bd)
    return qa.lib().qwen_hip_paged_attention_window(C.byref(a), C.byref(b), *d.values(), None)


def tree(qa, kvd={}, bd={}, **k):
    d = dict(out=P, q=P + 4096, dtype=qa.ST_F32, heads=4, scale=0.1, tree=P, words=1, ws=P, ws_bytes=1 << 40)
    d.update(k)
    a, b = kv(qa, **kvd), batch(qa, **bd)
    return qa.lib().qwen_hip_paged_attention_tree(C.byref(a), C.byref(b), *d.values(), None)


def append_at(qa, kvd={}, bd={}, **k):
    d = dict(rope_pos=P, q_out=P, q=P, k=P, v=P, dtype=qa.ST_F32, q_stride=512, kv_stride=256, heads=4, q_norm=P, k_norm=P,
             eps=1e-6, cos=P, sin=P, n_pos=64)
    d.update(k)
    a, b = kv(qa, **kvd), batch(qa, **bd)
    return qa.lib().qwen_hip_paged_append_at(C.byref(a), C.byref(b), *d.values(), None)


SINGLE = dict(row_start=None, rows=2)


@pytest.mark.parametrize("bad", BAD_KV)
def test_cache_refused(qa, bad):
    assert append_at(qa, kvd=bad) == EINVAL and "paged_append_at" in qa.last_error()
    assert tree(qa, kvd=bad) == EINVAL and "paged_attention_tree" in qa.last_error()
    for bd in ({}, SINGLE):
        assert window(qa, kvd=bad, bd=bd) == EINVAL and "paged_attention_window" in qa.last_error()


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_batch_refused(qa, bad):
    assert append_at(qa, bd=bad) == EINVAL
    assert tree(qa, bd=bad) == EINVAL
    assert window(qa, bd=bad) == EINVAL
    assert window(qa, bd=dict(SINGLE, **bad)) == EINVAL


BAD = [dict(dtype=1), dict(out=None), dict(q=None), dict(out=P + 4), dict(q=P + 8), dict(q=P), dict(heads=0), dict(heads=5),
       dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)]


@pytest.mark.parametrize("bad", BAD + [dict(window=0), dict(window=-1), dict(window=-2 ** 31), dict(sinks=-1)])
def test_window_refused(qa, bad):
    assert window(qa, **bad) == EINVAL
    assert "paged_attention_window" in qa.last_error()


@pytest.mark.parametrize("bad", BAD + [dict(tree=None), dict(tree=P + 4), dict(words=0), dict(words=-1), dict(words=5),
                                       dict(words=2 ** 31 - 1)])
def test_tree_refused(qa, bad):
    assert tree(qa, **bad) == EINVAL
    assert "paged_attention_tree" in qa.last_error()


@pytest.mark.parametrize("bad", [dict(rope_pos=None), dict(cos=None, sin=None), dict(cos=None), dict(q=None), dict(q_stride=508),
                                 dict(kv_stride=257), dict(n_pos=-1), dict(eps=-1.0), dict(q_norm=None)])
def test_append_at_refused(qa, bad):
    assert append_at(qa, **bad) == EINVAL
    assert "paged_append_at" in qa.last_error()


def test_single_rows(qa):
    """without row_start a sequence has one row"""
    assert window(qa, bd=dict(row_start=None, rows=3)) == EINVAL
    assert tree(qa, bd=dict(row_start=None, rows=3)) == EINVAL


def need(qa, what, kvd, bd, heads, *more):
    a, b = kv(qa, **kvd), batch(qa, **bd)
    return getattr(qa.lib(), "qwen_hip_paged_attention_%sws_bytes" % what)(C.byref(a), C.byref(b), heads, *more)


def test_workspace_refused(qa):
    """a call that splits its keys says how much it needs and takes no less"""
    kvd = dict(table_stride=4096)
    for bd in ({"rows": 2}, SINGLE):
        n = need(qa, "window_", kvd, bd, 4, 2000, 4)
        assert n > 0
        for bad in (dict(ws=None), dict(ws_bytes=n - 1), dict(ws=P + 4)):
            assert window(qa, kvd=kvd, bd=bd, window=2000, **bad) == EINVAL
            assert "workspace" in qa.last_error()
        n = need(qa, "tree_", kvd, bd, 4)
        assert n > 0
        for bad in (dict(ws=None), dict(ws_bytes=n - 1), dict(ws=P + 4)):
            assert tree(qa, kvd=kvd, bd=bd, **bad) == EINVAL
            assert "workspace" in qa.last_error()


def test_no_workspace_size_of_no_call(qa):
    L = qa.lib()
    assert L.qwen_hip_paged_attention_window_ws_bytes(None, None, 4, 10, 0) == 0
    assert L.qwen_hip_paged_attention_tree_ws_bytes(None, None, 4) == 0
    kvd = dict(table_stride=4096)
    assert need(qa, "window_", kvd, {"rows": 2}, 4, 0, 0) == need(qa, "window_", kvd, {"rows": 2}, 4, 5, -1) == 0


def test_workspace_bound(qa):
    """the size that serves every batch serves these as well"""
    rng, most = random.Random(2), 0
    for i in range(30000):
        kv_heads = rng.choice([1, 1, 2, 3, 5, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 9, 16, 64])
        n_seqs = min(int(2 ** rng.uniform(0, 14)), (1 << 20) // heads)
        packed = rng.random() < 0.6
        rows = max(1, min(int(2 ** rng.uniform(0, 17)), (1 << 23) // heads)) if packed else n_seqs
        kvd = dict(n_seqs=n_seqs, kv_heads=kv_heads, dtype=rng.choice([qa.ST_F32, qa.ST_BF16]), page_size=rng.choice([1, 16, 64]),
                   table_stride=1 << 16, n_pages=64)
        bd = dict(rows=rows, max_len=int(2 ** rng.uniform(0, 20)), row_start=P if packed else None)
        most = max(most, need(qa, "tree_", kvd, bd, heads),
                   need(qa, "window_", kvd, bd, heads, int(2 ** rng.uniform(0, 31)) - 1 or 1, int(2 ** rng.uniform(0, 31)) - 1))
    assert 0 < most <= qa.PAGED_ATTENTION_WS_MAX


def test_no_rows_is_no_call(qa):
    none = dict(k=None, v=None, table=None)
    for bd, kvd in ((dict(rows=0), none), (dict(rows=3), dict(none, n_seqs=0))):
        assert window(qa, kvd=kvd, bd=bd) == 0
        assert tree(qa, kvd=kvd, bd=bd, tree=None) == 0
        assert append_at(qa, kvd=kvd, bd=bd, rope_pos=None) == 0

"""Refusals of the paged cache's and the token drawing's entry points: everything the host can see
is checked before anything is launched, so these run without a GPU (the pointers are never read)."""
import ctypes as C
import math
import random

import pytest

EINVAL = -1
P = 0x10000        # 16-byte aligned, never read


def kv(qa, **k):
    d = dict(k=P, v=P, table=P, dtype=qa.ST_BF16, n_pages=4, page_size=16, kv_heads=2, head_dim=128, n_seqs=2,
             table_stride=2)
    d.update(k)
    return qa.PagedKV(*[d[n] for n, _ in qa.PagedKV._fields_])


def batch(qa, **k):
    d = dict(row_start=P, kv_len=P, rows=5, max_len=0)
    d.update(k)
    return qa.PagedBatch(*[d[n] for n, _ in qa.PagedBatch._fields_])


def append(qa, kvd={}, bd={}, **k):
    d = dict(q_out=P, q=P, k=P, v=P, dtype=qa.ST_F32, q_stride=512, kv_stride=256, heads=4, q_norm=P, k_norm=P,
             eps=1e-6, cos=P, sin=P, n_pos=64)
    d.update(k)
    a, b = kv(qa, **kvd), batch(qa, **bd)
    return qa.lib().qwen_hip_paged_append(C.byref(a), C.byref(b), *d.values(), None)


def attend(qa, which, kvd={}, bd={}, **k):
    d = dict(out=P, q=P + 4096, dtype=qa.ST_F32, heads=4, scale=0.1, ws=P, ws_bytes=1 << 40)
    d.update(k)
    a, b = kv(qa, **kvd), batch(qa, **bd)
    return getattr(qa.lib(), "qwen_hip_paged_attention_" + which)(C.byref(a), C.byref(b), *d.values(), None)


BAD_KV = [dict(dtype=1), dict(dtype=-1), dict(head_dim=64), dict(page_size=0), dict(page_size=24),
          dict(page_size=1 << 25), dict(n_pages=0), dict(kv_heads=0), dict(kv_heads=3), dict(n_seqs=-1), dict(n_pages=2 ** 31 - 1),
          dict(table_stride=0), dict(k=None), dict(v=None), dict(table=None), dict(k=P + 8), dict(v=P + 2)]
BAD_BATCH = [dict(rows=-1), dict(max_len=-1), dict(kv_len=None), dict(rows=2 ** 31 - 1)]


@pytest.mark.parametrize("bad", BAD_KV)
def test_cache_refused(qa, bad):
    assert append(qa, kvd=bad) == EINVAL and "paged_append" in qa.last_error()
    assert attend(qa, "prefill", kvd=bad) == EINVAL and "prefill" in qa.last_error()
    assert attend(qa, "decode", kvd=bad, bd=dict(row_start=None, rows=2)) == EINVAL and "decode" in qa.last_error()


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_batch_refused(qa, bad):
    assert append(qa, bd=bad) == EINVAL
    assert attend(qa, "prefill", bd=bad) == EINVAL
    assert attend(qa, "decode", bd=dict(dict(row_start=None, rows=2), **bad)) == EINVAL


@pytest.mark.parametrize("bad", [dict(dtype=1), dict(q_out=None), dict(q=None), dict(k=None), dict(v=None),
                                 dict(q_out=P + 4), dict(k=P + 8), dict(q_stride=508), dict(q_stride=513),
                                 dict(kv_stride=128), dict(kv_stride=257), dict(heads=0), dict(heads=3),
                                 dict(q_norm=None), dict(k_norm=None), dict(cos=None), dict(sin=None),
                                 dict(sin=P + 4), dict(eps=-1.0), dict(eps=math.nan), dict(n_pos=-1),
                                 dict(q_stride=516)])
def test_append_refused(qa, bad):
    assert append(qa, **bad) == EINVAL
    assert "paged_append" in qa.last_error()


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("bad", [dict(dtype=1), dict(out=None), dict(q=None), dict(out=P + 4), dict(q=P + 8),
                                 dict(q=P), dict(heads=0), dict(heads=5), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=math.inf), dict(scale=math.nan)])
def test_attention_refused(qa, which, bad):
    bd = dict(row_start=None, rows=2) if which == "decode" else {}
    assert attend(qa, which, bd=bd, **bad) == EINVAL
    assert which in qa.last_error()


def test_attention_refuses_the_other_ones_batch(qa):
    assert attend(qa, "prefill", bd=dict(row_start=None, rows=2)) == EINVAL
    assert attend(qa, "decode", bd=dict(rows=2)) == EINVAL
    assert attend(qa, "decode", bd=dict(row_start=None, rows=3)) == EINVAL      # one row per sequence
    assert append(qa, bd=dict(row_start=None, rows=3)) == EINVAL


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_attention_workspace_refused(qa, which):
    """a call that splits its keys says how much it needs and takes no less"""
    kvd = dict(table_stride=4096)
    bd = dict(row_start=None if which == "decode" else P, rows=2)
    a, b = kv(qa, **kvd), batch(qa, **bd)
    need = qa.lib().qwen_hip_paged_attention_ws_bytes(C.byref(a), C.byref(b), 4)
    assert need > 0
    for bad in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=P + 4)):
        assert attend(qa, which, kvd=kvd, bd=bd, **bad) == EINVAL
        assert "workspace" in qa.last_error()


def ws_bytes(qa, rows, n_seqs, heads, kv_heads, max_len, dtype, page, packed):
    a = kv(qa, n_seqs=n_seqs, kv_heads=kv_heads, dtype=dtype, page_size=page, table_stride=1 << 16, n_pages=64)
    b = batch(qa, rows=rows, max_len=max_len, row_start=P if packed else None)
    return qa.lib().qwen_hip_paged_attention_ws_bytes(C.byref(a), C.byref(b), heads)


def test_attention_workspace_bound(qa):
    """one size for all batches: the need does not grow with the batch (a smaller one is split further)"""
    need = [ws_bytes(qa, rows, 8, 16, 8, 4096, qa.ST_BF16, 64, True) for rows in (8000, 4000, 2500, 2000, 512)]
    assert need[0] == 0 and need[2] > need[4] > 0
    most, rng = {True: 0, False: 0}, random.Random(1)
    for i in range(60000):
        kv_heads = rng.choice([1, 1, 2, 3, 5, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 9, 16, 64])
        n_seqs = min(int(2 ** rng.uniform(0, 14)), (1 << 20) // heads)
        packed = rng.random() < 0.6
        # around the borders of the plans as well
        near = rng.choice([128, 64]) * rng.randint(1, 400) + rng.choice([-1, 0, 1]) if rng.random() < 0.5 else int(2 ** rng.uniform(0, 17))
        rows = max(1, min(near, (1 << 23) // heads)) if packed else n_seqs
        most[packed] = max(most[packed], ws_bytes(qa, rows, n_seqs, heads, kv_heads, int(2 ** rng.uniform(0, 20)),
                                                  rng.choice([qa.ST_F32, qa.ST_BF16]), rng.choice([1, 16, 64]), packed))
    # below it, and not by much
    assert qa.PAGED_ATTENTION_WS_MAX / 2 < most[True] <= qa.PAGED_ATTENTION_WS_MAX
    assert qa.PAGED_ATTENTION_WS_MAX / 8 < most[False] <= qa.PAGED_ATTENTION_WS_MAX


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_blocks_than_a_launch_has_refused(qa, dtype):
    """sequences without rows have a block a kv head all the same: more than 2^32 threads are no launch"""
    kvd = dict(n_seqs=1 << 22, kv_heads=8, dtype=qa.ST_F32 if dtype == "f32" else qa.ST_BF16)
    assert attend(qa, "prefill", kvd=kvd, bd=dict(rows=1), heads=8) == EINVAL
    assert "qk_paged_prefill_launch" in qa.last_error()


def test_no_rows_is_no_call(qa):
    """no rows: nothing to launch, whatever the pointers"""
    none = dict(k=None, v=None, table=None)
    assert append(qa, kvd=none, bd=dict(rows=0)) == 0
    assert attend(qa, "prefill", kvd=none, bd=dict(rows=0)) == 0
    assert attend(qa, "decode", kvd=dict(none, n_seqs=0), bd=dict(rows=0, row_start=None)) == 0
    assert sample(qa, rows=0, tokens=None, logits=None) == 0
    assert qa.lib().qwen_hip_paged_attention_ws_bytes(None, None, 4) == 0


def test_no_sequences_is_no_call(qa):
    """rows of no sequence are left as they are; row_start has one entry then"""
    for k in (dict(kvd=dict(n_seqs=0), bd=dict(rows=3)), dict(kvd=dict(n_seqs=0), bd=dict(rows=500))):
        assert append(qa, **k) == 0
        assert attend(qa, "prefill", **k) == 0


@pytest.mark.parametrize("rows", [1, 3, 31, 63, 500])
@pytest.mark.parametrize("heads,dtype", [(2, "f32"), (4, "f32"), (4, "bf16"), (16, "bf16")])
def test_no_sequences_need_no_workspace(qa, rows, heads, dtype):
    """the size that a program asks for before such a call"""
    a, b = kv(qa, n_seqs=0, dtype=qa.ST_F32 if dtype == "f32" else qa.ST_BF16, table_stride=4096), batch(qa, rows=rows)
    assert qa.lib().qwen_hip_paged_attention_ws_bytes(C.byref(a), C.byref(b), heads) == 0
    assert attend(qa, "prefill", kvd=dict(n_seqs=0, table_stride=4096), bd=dict(rows=rows), heads=heads, ws=None, ws_bytes=0) == 0


def sample(qa, **k):
    d = dict(tokens=P, logits=P, row_stride=1000, rows=2, vocab=1000, temperature=P, top_k=P, top_p=P, min_p=P, u=P,
             ws=P, ws_bytes=1 << 40)
    d.update(k)
    return qa.lib().qwen_hip_sample(*d.values(), None)


@pytest.mark.parametrize("bad", [dict(tokens=None), dict(logits=None), dict(u=None), dict(ws=None), dict(ws=P + 4),
                                 dict(ws_bytes=0), dict(row_stride=999), dict(rows=-1), dict(rows=(1 << 16) + 1),
                                 dict(vocab=0), dict(vocab=(1 << 20) + 1, row_stride=1 << 21)])
def test_sample_refused(qa, bad):
    assert sample(qa, **bad) == EINVAL
    assert "sample" in qa.last_error()


def test_sample_workspace_bytes(qa):
    ws = qa.lib().qwen_hip_sample_ws_bytes
    assert ws(2, 1000) > 0 and ws(64, 151936) >= 64 * ws(1, 151936)
    assert ws(0, 10) == ws(-1, 10) == ws(1, 0) == ws(1, (1 << 20) + 1) == ws((1 << 16) + 1, 10) == 0
    assert sample(qa, ws_bytes=ws(2, 1000) - 1) == EINVAL

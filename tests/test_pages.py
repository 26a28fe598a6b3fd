"""Refusals of page tables that continue others, copies, accepted drafts and beam selection: what the host can see is
checked before anything is launched (no GPU, the pointers are never read)."""
import ctypes as C

import pytest

from test_paged import BAD_KV, EINVAL, P, batch, kv

Q = 0x4000000          # apart from P by more than any buffer here


def layers(qa, n=2, **k):
    return (qa.PagedKV * n)(*[kv(qa, **k) for _ in range(n)])


def fork(qa, kvd={}, **k):
    d = dict(kv_len=P, parent=P, new_rows=P, outside=P, n_out=3, table_out=Q, len_out=Q + 4096, copies=Q + 8192, missing=Q,
             ws=None, ws_bytes=0)
    d.update(k)
    a = kv(qa, **kvd)
    return qa.lib().qwen_hip_paged_fork(C.byref(a), *d.values(), None)


def copy(qa, kvd={}, change=None, n_layers=2, **k):
    d = dict(copies=P, n_copies=4)
    d.update(k)
    a = layers(qa, 2, **kvd)
    for n, v in (change or {}).items():
        setattr(a[1], n, v)
    return qa.lib().qwen_hip_paged_copy(a, n_layers, *d.values(), None)


def compact(qa, kvd={}, bd={}, change=None, n_layers=2, **k):
    d = dict(len_out=Q, path=P, path_stride=8, n_path=P)
    d.update(k)
    a, b = layers(qa, 2, **kvd), batch(qa, **bd)
    for n, v in (change or {}).items():
        setattr(a[1], n, v)
    return qa.lib().qwen_hip_paged_compact(a, n_layers, C.byref(b), *d.values(), None)


def beam(qa, **k):
    d = dict(parent=P, token=P, score_out=P, logits=P, dtype=qa.ST_F32, row_stride=1000, seqs=2, beams=4, vocab=1000, score=Q,
             ended=Q + 0x10000, n_out=8, ws=P, ws_bytes=1 << 40)
    d.update(k)
    return qa.lib().qwen_hip_beam_select(*d.values(), None)


@pytest.mark.parametrize("bad", BAD_KV)
def test_cache_refused(qa, bad):
    heads = bad == dict(kv_heads=3)                        # no refusal here: no query heads to share it
    if "k" not in bad and "v" not in bad and not heads:
        assert fork(qa, kvd=bad) == EINVAL and "paged_fork" in qa.last_error()
    if "table" not in bad and "n_seqs" not in bad and "table_stride" not in bad and not heads:
        assert copy(qa, kvd=bad) == EINVAL and "paged_copy" in qa.last_error()
    if not heads:
        assert compact(qa, kvd=bad) == EINVAL and "paged_compact" in qa.last_error()


@pytest.mark.parametrize("bad", [dict(n_out=-1), dict(n_out=1025), dict(kv_len=None), dict(table_out=None), dict(len_out=None),
                                 dict(copies=None), dict(copies=Q + 8), dict(missing=None), dict(parent=None), dict(table_out=P),
                                 dict(table_out=P + 12), dict(table_out=P - 20), dict(len_out=P), dict(len_out=P + 4),
                                 dict(len_out=P - 8)])
def test_fork_refused(qa, bad):
    assert fork(qa, **bad) == EINVAL
    assert "paged_fork" in qa.last_error()


def test_fork_workspace(qa):
    L = qa.lib()
    def need(n_pages, n_out=3):
        a = kv(qa, n_pages=n_pages, page_size=1)
        return L.qwen_hip_paged_fork_ws_bytes(C.byref(a), n_out)
    assert need(1 << 19) == 0 and need(1 << 19, 1024) == 0
    n = need((1 << 19) + 1)
    assert n >= 2 * ((1 << 19) + 1) // 8
    assert fork(qa, kvd=dict(table_stride=1 << 30)) == EINVAL and "page ids" in qa.last_error()
    assert need((1 << 19) + 1, 0) == need((1 << 19) + 1, 1025) == L.qwen_hip_paged_fork_ws_bytes(None, 1) == 0
    big = dict(n_pages=(1 << 19) + 1, page_size=1)
    for bad in (dict(ws=None, ws_bytes=n), dict(ws=Q, ws_bytes=n - 1), dict(ws=Q + 4, ws_bytes=n)):
        assert fork(qa, kvd=big, **bad) == EINVAL and "workspace" in qa.last_error()


@pytest.mark.parametrize("bad", [dict(n_layers=0), dict(n_layers=-1), dict(n_layers=65), dict(n_copies=-1), dict(copies=None),
                                 dict(copies=P + 4), dict(n_copies=1 << 24)] +
                         [dict(change={n: v}) for n, v in (("dtype", 0), ("n_pages", 5), ("page_size", 8), ("kv_heads", 1),
                                                           ("head_dim", 64), ("k", None), ("v", None), ("v", P + 8))])
def test_copy_refused(qa, bad):
    assert copy(qa, **bad) == EINVAL
    assert "paged_copy" in qa.last_error() or "n_copies" in bad


@pytest.mark.parametrize("bad", [dict(n_layers=0), dict(n_layers=65), dict(len_out=None), dict(path=None), dict(n_path=None),
                                 dict(path_stride=0), dict(path_stride=-1), dict(len_out=P), dict(len_out=P + 4),
                                 dict(bd=dict(kv_len=None)), dict(bd=dict(rows=-1)), dict(bd=dict(row_start=None, rows=5)),
                                 dict(kvd=dict(table=None))] +
                         [dict(change={n: v}) for n, v in (("dtype", 0), ("n_pages", 5), ("page_size", 8), ("kv_heads", 1),
                                                           ("table", Q), ("table_stride", 3), ("n_seqs", 1), ("k", None))])
def test_compact_refused(qa, bad):
    assert compact(qa, **bad) == EINVAL
    assert "paged_compact" in qa.last_error()


def test_no_layers(qa):
    assert qa.lib().qwen_hip_paged_copy(None, 2, P, 1, None) == EINVAL
    b = batch(qa)
    assert qa.lib().qwen_hip_paged_compact(None, 2, C.byref(b), Q, P, 8, P, None) == EINVAL
    a = layers(qa, 1)
    assert qa.lib().qwen_hip_paged_compact(a, 1, None, Q, P, 8, P, None) == EINVAL


def test_nothing_is_no_call(qa):
    assert fork(qa, n_out=0, table_out=None) == 0
    assert copy(qa, n_copies=0, copies=None) == 0
    assert compact(qa, kvd=dict(n_seqs=0), len_out=None) == 0
    assert beam(qa, seqs=0, logits=None) == 0


@pytest.mark.parametrize("bad", [dict(seqs=-1), dict(beams=0), dict(beams=65), dict(beams=-1), dict(vocab=0),
                                 dict(vocab=(1 << 20) + 1, row_stride=1 << 21), dict(n_out=0), dict(n_out=65),
                                 dict(seqs=(1 << 14) + 1), dict(seqs=2 ** 31 - 1), dict(dtype=1), dict(dtype=-1), dict(row_stride=999),
                                 dict(row_stride=-1000), dict(parent=None), dict(token=None), dict(score_out=None),
                                 dict(logits=None), dict(score=None), dict(logits=P + 2), dict(ws=None), dict(ws=P + 4),
                                 dict(ws_bytes=0), dict(score_out=Q - 8), dict(score_out=Q + 28), dict(parent=Q), dict(token=Q),
                                 dict(parent=Q + 0x10000 - 60), dict(token=Q + 0x10000), dict(score_out=Q + 0x10000 + 31)])
def test_beam_refused(qa, bad):
    assert beam(qa, **bad) == EINVAL
    assert "beam_select" in qa.last_error()


def test_beam_workspace_bytes(qa):
    ws = qa.lib().qwen_hip_beam_select_ws_bytes
    assert ws(2, 4, 1000, 8) > 0
    assert ws(0, 4, 10, 4) == ws(1, 0, 10, 4) == ws(1, 65, 10, 4) == ws(1, 4, 0, 4) == ws(1, 4, 10, 0) == ws(1, 4, 10, 65) == 0
    assert ws(1 << 10, 64, 1 << 20, 64) > 1 << 32
    assert beam(qa, ws_bytes=ws(2, 4, 1000, 8) - 1) == EINVAL

"""Outputs that overlap what other blocks or threads of the same launch still read are refused (no GPU, the pointers are
never read)."""
import pytest

from test_pages import EINVAL, P, Q, compact, fork

# apart from each other: a table of 2 rows of 2, lengths, rows of 3 new sequences, a byte for each of 4 pages
IN = dict(parent=P + 0x1000, new_rows=P + 0x2000, outside=P + 0x3000)
OUT = dict(table_out=Q, len_out=Q + 0x1000, copies=Q + 0x2000, missing=Q + 0x3000)


@pytest.mark.parametrize("bad", [dict(copies=IN["parent"]), dict(copies=IN["new_rows"] - 32), dict(copies=IN["outside"]),
                                 dict(copies=P), dict(len_out=IN["parent"] + 4), dict(len_out=IN["parent"] - 8),
                                 dict(len_out=IN["new_rows"] + 8), dict(len_out=IN["outside"]), dict(len_out=IN["outside"] - 8),
                                 dict(table_out=IN["outside"] - 20), dict(table_out=IN["outside"]),
                                 dict(table_out=IN["parent"]), dict(table_out=IN["new_rows"] + 8), dict(missing=IN["outside"]),
                                 dict(missing=IN["parent"] + 8), dict(missing=IN["new_rows"]), dict(missing=P)])
def test_fork(qa, bad):
    assert fork(qa, **{**IN, **OUT, **bad}) == EINVAL
    assert "paged_fork" in qa.last_error() and "overlap" in qa.last_error()


@pytest.mark.parametrize("bad", [dict(n_path=Q), dict(n_path=Q - 4), dict(n_path=Q + 4), dict(path=Q), dict(path=Q - 40),
                                 dict(path=Q + 4), dict(bd=dict(row_start=Q)), dict(bd=dict(row_start=Q - 8)),
                                 dict(bd=dict(row_start=Q + 4)), dict(kvd=dict(table=Q - 12))])
def test_compact(qa, bad):
    """2 sequences: row starts of 3, paths 8 entries apart, a table of 4"""
    assert compact(qa, **bad) == EINVAL
    assert "paged_compact" in qa.last_error() and "overlap" in qa.last_error()

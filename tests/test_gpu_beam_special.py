"""Logits that are no number: each such row is a sequence of one beam, or the beam whose candidates come first,
so that what it gives is what is compared (tests/pages_util.py has the definition)."""
import math

import pytest
import torch as T

from pages_util import beam, check_beam

pytestmark = pytest.mark.gpu

DT = {"f32": T.float32, "bf16": T.bfloat16}
# quiet and signalling, both signs, the smallest and the largest payload
NANS = {"f32": [0x7fc00000, 0xffc00000, 0x7f800001, 0xff800001, 0x7fffffff, 0xffffffff],
        "bf16": [0x7fc0, 0xffc0, 0x7f81, 0xff81, 0x7fff, 0xffff]}
# shares of 8, 16 and 32 entries a thread, whole and ragged
SHAPES = [(1, 1), (7, 4), (300, 64), (2049, 16), (9001, 17), (151936, 4), (151936, 64)]


def normal(seed, rows, vocab, dtype, spread=2.0):
    g = T.Generator().manual_seed(seed)
    return (T.randn(rows, vocab, generator=g) * spread).to(DT[dtype])


def put(x, row, at, bits):
    """the value of these bits, as they are"""
    width, kind = (32, T.int32) if x.dtype == T.float32 else (16, T.int16)
    x.view(kind)[row, at] = bits - (1 << width) if bits >> (width - 1) else bits


def positions(vocab):
    """the first, the last, and ones in the shares' inner and last planes"""
    return sorted({0, vocab - 1, vocab // 2, vocab // 3, max(vocab - 2, 0), min(2047, vocab - 1)})


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,n_out", SHAPES)
def test_one_entry_that_is_no_number(qa, gpu, dtype, vocab, n_out):
    """the choice is that of the same row with -infinity there, score and all"""
    at = positions(vocab)
    x = normal(vocab, len(at) * len(NANS[dtype]), vocab, dtype)
    y = x.clone()
    for i in range(x.shape[0]):
        put(x, i, at[i // len(NANS[dtype])], NANS[dtype][i % len(NANS[dtype])])
        y[i, at[i // len(NANS[dtype])]] = -math.inf
    score = [-0.25 * i for i in range(x.shape[0])]
    x, y = x.cuda(), y.cuda()
    got = beam(qa, x, score, None, n_out, x.shape[0])
    if vocab <= 9001:
        check_beam(got, x, score, None, x.shape[0])
    for a, b in zip(got, beam(qa, y, score, None, n_out, x.shape[0])):
        assert (a == b).all()
    if vocab == 1:
        assert (got[0] == -1).all() and (got[1] == -1).all() and (got[2] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,n_out", SHAPES)
def test_rows_of_no_numbers(qa, gpu, dtype, vocab, n_out):
    """no entry is one: no candidates; some are: these, and the logarithm over these"""
    for k, bits in enumerate(NANS[dtype] if vocab <= 9001 else NANS[dtype][1:4:2]):
        x = normal(k, 4, vocab, dtype)
        for at in range(0, vocab, 2):
            put(x, 1, at, bits)
        put(x, 0, slice(None), bits)
        put(x, 2, slice(0, vocab - 1), bits)
        put(x, 3, slice(None), bits)
        x[3, vocab // 2] = -math.inf
        x = x.cuda()
        score = [-1.0, -2.0, -3.0, -4.0]
        got = beam(qa, x, score, None, n_out, 4)
        check_beam(got, x, score, None, 4)
        parent, token, out = got
        for q in (0, 3):
            assert (parent[q] == -1).all() and (token[q] == -1).all() and (out[q] == -math.inf).all()
        assert all(t % 2 for t in token[1] if t >= 0)
        assert token[2, 0] == vocab - 1 and abs(out[2, 0] + 3.0) <= 2.0 ** -22 and (token[2, 1:] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("beams,n_out", [(2, 2), (8, 16), (40, 64)])
def test_such_beams_among_others(qa, gpu, dtype, beams, n_out):
    """the beam with entries that are no number is the best by far: its own candidates come first, then the others'"""
    vocab = 5003
    for k, bits in enumerate(NANS[dtype]):
        x = normal(k, beams, vocab, dtype, 0.5)
        score = [-30.0 - 0.01 * b for b in range(beams)]
        b = beams // 2
        score[b] = 0.0
        score = T.tensor(score).tolist()                   # as the call takes them: in fp32
        finite = [4, 1001, 1002, 4090, 5001]
        keep = x[b, finite].clone()
        put(x, b, slice(None), bits)
        x[b, finite] = keep
        x = x.cuda()
        got = beam(qa, x, score, None, n_out, 1)
        check_beam(got, x, score, None, 1)
        n = min(n_out, 5)
        assert (got[0][0, :n] == b).all() and set(got[1][0, :n].tolist()) <= set(finite)
        assert (got[0][0, n:] != b).all()
        # ... and one without a number at all has none of the places
        y = x.cpu()
        put(y, b, slice(None), bits)
        y = y.cuda()
        got = beam(qa, y, score, None, n_out, 1)
        check_beam(got, y, score, None, 1)
        assert (got[0] != b).all() and (got[0] >= 0).all()

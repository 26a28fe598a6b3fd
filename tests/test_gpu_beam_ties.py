"""Candidates whose scores are equal in 64 bits: by row, by falling logit, by token."""
import math

import numpy as np
import pytest
import torch as T

from pages_util import T as DT, beam, beam_scores, clean

pytestmark = pytest.mark.gpu

LOW = float(np.finfo(np.float32).min)
# few and many places: bounds by counting, by the waves' largest, by steps
SHAPES = [(1, 3), (50, 64), (300, 16), (2049, 16), (9001, 17), (40000, 4), (151936, 64)]


def normal(seed, rows, vocab, dtype, spread=2.0):
    g = T.Generator().manual_seed(seed)
    return (T.randn(rows, vocab, generator=g) * spread).to(DT[dtype])


def check(qa, x, score, ended, n_out, seqs):
    """the definition's order throughout, and its scores: as fp32 holds them, but for 2^-22 of the row's logarithm"""
    got = beam(qa, x.cuda(), score, ended, n_out, seqs)
    x = x.double().numpy()
    B = x.shape[0] // seqs
    for q in range(seqs):
        rows = slice(q * B, (q + 1) * B)
        s = beam_scores(x[rows], score[rows], None if ended is None else ended[rows])
        b, t = np.nonzero(s > -math.inf)
        key = s[b, t]
        order = np.lexsort((t, -clean(x[rows])[b, t], b, -key))[:n_out]
        n = len(order)
        assert got[0][q, :n].tolist() == (q * B + b[order]).tolist() and got[1][q, :n].tolist() == t[order].tolist()
        assert (got[0][q, n:] == -1).all() and (got[1][q, n:] == -1).all() and (got[2][q, n:] == -math.inf).all()
        with np.errstate(over="ignore"):
            want = key[order].astype(np.float32).astype(np.float64)
        same = got[2][q, :n].astype(np.float64) == want
        assert (same | (np.abs(got[2][q, :n] - key[order]) <= 2.0 ** -22 + 2.0 ** -24 * np.abs(key[order]))).all()
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,n_out", SHAPES)
def test_scores_that_hide_the_logits(qa, gpu, dtype, vocab, n_out):
    """a beam that should not be used has a score so low (or one so high) that all its tokens have the same one"""
    score = [-1e30, LOW, 1e30, -LOW, -1e20]
    x = normal(vocab, 5, vocab, dtype)
    x[:, ::7] = -math.inf
    x[:, vocab - 1] = 1.0
    got = check(qa, x, score, None, n_out, 5)
    best = T.sort(x[0].float(), descending=True, stable=True)[1][:n_out].tolist()
    n = min(n_out, int((x[0] > -math.inf).sum()))
    assert got[1][0, :n].tolist() == best[:n]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,n_out", SHAPES[1:])
def test_scores_that_hide_near_logits(qa, gpu, dtype, vocab, n_out):
    """beside -1e9 what is left of a logit is 2^-23: of the entries within that, the larger ones first"""
    x = normal(vocab, 2, vocab, dtype, 1e-7)
    x[1] = 3.0
    x[1, ::5] += 1e-6
    got = beam(qa, x.cuda(), [-1e9, -1e9], None, n_out, 2)
    for q in range(2):
        want = T.sort(x[q].float(), descending=True, stable=True)[1][:n_out].tolist()
        assert got[1][q].tolist()[:len(want)] == want and got[1][q].tolist()[len(want):] == [-1] * (n_out - len(want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("beams,n_out,vocab", [(4, 4, 151936), (8, 16, 5003), (64, 64, 5003), (64, 64, 3), (33, 48, 1), (12, 24, 30011)])
def test_hidden_beams(qa, gpu, dtype, beams, n_out, vocab):
    """one beam counts and has few candidates, the others' scores are as low as that: their places by row and logit"""
    x = normal(beams, beams, vocab, dtype)
    score = [-1e30] * beams
    live = beams // 2
    score[live] = -3.0
    x[live, 2:] = -math.inf
    got = check(qa, x, score, None, n_out, 1)
    assert (got[0][0, :min(2, vocab)] == live).all()
    # ... at steps of each other; and all alike
    check(qa, x, [-1e30 if b % 3 else -2e30 for b in range(beams)], None, n_out, 1)
    check(qa, x, [-1e30] * beams, None, n_out, 1)
    ended = [b % vocab if b % 4 == 1 else -1 for b in range(beams)]
    check(qa, x, [-1e30] * beams, ended, n_out, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,n_out", SHAPES[2:])
def test_infinite_entries(qa, gpu, dtype, vocab, n_out):
    """+infinity is the largest number, whichever entry has it, beside which no other logit counts; -infinity is none"""
    x = normal(3, 5, vocab, dtype)
    big = T.finfo(T.float32).max if dtype == "f32" else math.inf
    x[0, 17], x[0, vocab - 1], x[0, 5] = math.inf, math.inf, big
    x[1] = -math.inf
    x[1, vocab - 1], x[1, 3] = 3.0, math.inf
    x[2] = -math.inf
    x[2, vocab - 2] = 3.0
    x[3] = math.inf
    x[4] = T.where(T.rand(vocab, generator=T.Generator().manual_seed(4)) < 0.99, -math.inf, 1.0).to(DT[dtype])
    score = [-1.0, -2.0, -3.0, -4.0, -5.0]
    got = check(qa, x, score, None, n_out, 5)
    n = min(n_out, 3)
    assert got[1][0, :n].tolist() == [5, 17, vocab - 1][:n] and (got[1][1, 0], got[1][2, 0]) == (3, vocab - 2)
    assert got[1][3].tolist() == list(range(n_out))
    check(qa, x[1:], score[1:], None, n_out, 2)
def test_scores_below_the_numbers(qa, gpu):
    """what is below fp32's numbers is written as -infinity, behind all others, by row and token as it is"""
    low = float(np.finfo(np.float32).min)
    x = T.full((2, 40), low)
    x[0, 7], x[1, 9] = 1.0, 2.0
    x, score = x.cuda(), [-2.0, low]
    parent, token, out = beam(qa, x, score, None, 64, 1)
    s = beam_scores(x.double().cpu().numpy(), score, None).ravel()
    order = np.argsort(-s, kind="stable")[:64]
    assert parent[0].tolist() == (order // 40).tolist() and token[0].tolist() == (order % 40).tolist()
    assert (out[0, :41] >= low).all() and (out[0, 41:] == -math.inf).all()

"""The choice of the best continuations over beams and vocabulary, through the C ABI on device memory, against the
definition in 64 bits (tests/pages_util.py)."""
import math

import numpy as np
import pytest
import torch as T

from pages_util import beam, beam_scores, check_beam

pytestmark = pytest.mark.gpu

DT = {"f32": T.float32, "bf16": T.bfloat16}


def inputs(seed, rows, vocab, dtype="f32", spread=2.0):
    g = T.Generator().manual_seed(seed)
    x = (T.randn(rows, vocab, generator=g) * spread).to(DT[dtype]).cuda()
    return x, (-20 * T.rand(rows, generator=g)).tolist(), g


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 151, 1024, 2047, 2048, 2049, 8191, 8193, 16384, 50001])
@pytest.mark.parametrize("beams,n_out", [(1, 1), (4, 4), (3, 17), (8, 16), (2, 64)])
def test_beam(qa, gpu, dtype, vocab, beams, n_out):
    """sizes around the shares' borders; more places than candidates"""
    x, score, _ = inputs(vocab + beams, 2 * beams, vocab, dtype)
    check_beam(beam(qa, x, score, None, n_out, 2), x, score, None, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs,beams,n_out", [(1, 4, 4), (8, 8, 16), (32, 1, 1), (1, 64, 64), (2, 20, 40)])
def test_beam_vocabulary(qa, gpu, dtype, seqs, beams, n_out):
    x, score, _ = inputs(seqs, seqs * beams, 151936, dtype, 3.0)
    check_beam(beam(qa, x, score, None, n_out, seqs), x, score, None, seqs)


@pytest.mark.parametrize("dtype,rows,seqs,n_out", [("f32", 3, 1, 64), ("bf16", 4, 2, 20), ("f32", 2, 2, 3)])
def test_beam_largest_vocabulary(qa, gpu, dtype, rows, seqs, n_out):
    x, score, _ = inputs(77, rows, 1 << 20, dtype)
    check_beam(beam(qa, x, score, None, n_out, seqs), x, score, None, seqs)


@pytest.mark.parametrize("n_out", [1, 7, 64])
def test_beam_many_like_candidates(qa, gpu, n_out):
    """thousands of candidates within a share's few: a list of them has to be cut more than once"""
    g = T.Generator().manual_seed(78)
    x = T.full((1, 5000), -30.0)
    x[:, ::3] = T.randint(0, 3, (1, 1667), generator=g).float() * 1e-6
    x = x.repeat(64, 1).cuda()                             # equal beams: which comes first is the definition's
    check_beam(beam(qa, x, [-1.0] * 64, None, n_out, 1), x, [-1.0] * 64, None, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("skew", [0, 1, 2, 3, 5, 7])
@pytest.mark.parametrize("pad", [0, 1, 13])
def test_beam_alignment(qa, gpu, dtype, skew, pad):
    """rows at any alignment to their type, any distance apart; what lies between them is infinite"""
    rows, vocab = 6, 5003
    x, score, _ = inputs(5, rows, vocab, dtype)
    wide = T.full((rows * (vocab + pad) + skew + 16,), math.inf, dtype=DT[dtype], device="cuda")
    v = wide[skew:skew + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab]
    v.copy_(x)
    check_beam(beam(qa, v, score, None, 9, 2), x, score, None, 2)


def test_beam_ended(qa, gpu):
    """beams at their end keep their score and give one candidate; ids outside the vocabulary are no end"""
    x, score, g = inputs(6, 24, 3001)
    ended = T.randint(-1, 3001, (24,), generator=g).tolist()
    for i in range(0, 24, 3):
        ended[i] = [-1, -7, 3001, 2 ** 31 - 1][i // 3 % 4]
    for i in range(16, 24):
        ended[i] = i                                       # a sequence whose beams are all at their end
    check_beam(beam(qa, x, score, ended, 10, 3), x, score, ended, 3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [0.0, -0.0, 5.0, -3e38, 3e38])
@pytest.mark.parametrize("vocab,beams,n_out", [(151936, 4, 8), (5000, 64, 64), (40, 3, 64), (30000, 8, 33)])
def test_beam_equal_logits(qa, gpu, dtype, value, vocab, beams, n_out):
    """all candidates of equal beams are equal: the first ones, by beam and token"""
    x = T.full((beams, vocab), value, dtype=DT[dtype], device="cuda")
    if value == -0.0:
        x[:, ::2] = 0.0
    score = [-1.5] * beams
    parent, token, out = beam(qa, x, score, None, n_out, 1)
    n = min(n_out, beams * vocab)
    flat = np.arange(n)
    assert parent[0, :n].tolist() == (flat // vocab).tolist() and token[0, :n].tolist() == (flat % vocab).tolist()
    want = -1.5 - math.log(vocab)
    assert bool((np.abs(out[0, :n] - want) <= 2.0 ** -22 + 2.0 ** -24 * abs(want)).all())
    assert (parent[0, n:] == -1).all() and (token[0, n:] == -1).all() and (out[0, n:] == -math.inf).all()


def test_beam_equal_beams(qa, gpu):
    """equal beams: each of the best tokens once a beam, the lower beam first"""
    x, _, _ = inputs(8, 1, 10007)
    x = x.repeat(6, 1).contiguous()
    parent, token, out = beam(qa, x, [-2.0] * 6, None, 30, 1)
    best = T.sort(x[0], descending=True, stable=True)[1][:5].tolist()
    assert token[0].tolist() == [t for t in best for _ in range(6)] and parent[0].tolist() == list(range(6)) * 5


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["rising", "falling", "one thread's", "lowest type"])
def test_beam_orders(qa, gpu, dtype, order):
    """logits in order; the large ones all in one thread's share; forbidden by the type's lowest value"""
    vocab = 40000
    x, score, g = inputs(9, 8, vocab, dtype)
    if order in ("rising", "falling"):
        x = T.sort(x.float(), dim=1, descending=order == "falling")[0].to(DT[dtype]).contiguous()
    elif order == "one thread's":
        for j in range(8):
            x[:, 1024 * j + 12:1024 * j + 16] += 30.0
            x[:, 2048 * j + 16:2048 * j + 24] += 31.0
    else:
        x[:, T.randperm(vocab, generator=g)[:vocab - 11].cuda()] = T.finfo(DT[dtype]).min
    for n in (5, 20, 64):
        check_beam(beam(qa, x, score, None, n, 2), x, score, None, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_beam_not_finite(qa, gpu, dtype):
    """rows of nothing, of NaN, with one entry, with +inf; scores of -inf, NaN, +inf"""
    vocab = 9001
    x, score, g = inputs(10, 40, vocab, dtype)
    ninf = -math.inf
    x[0] = ninf
    x[1] = math.nan
    x[2], x[2, 8999] = ninf, 3.0
    x[3, 17], x[3, 9000] = math.inf, math.inf
    x[4, ::2] = math.nan
    x[5] = T.where(T.rand(vocab, generator=g).cuda() < 0.999, ninf, 1.0).to(DT[dtype])
    x[8:16] = ninf                                         # a sequence without candidates
    score[17], score[18], score[19] = ninf, math.nan, math.inf
    for i in range(24, 32):
        score[i] = ninf                                    # the first step: all beams but one have no score
    score[24] = 0.0
    x[32:40] = ninf
    x[33, 5], x[36, 6], x[36, 4] = 1.0, 2.0, 2.0           # fewer candidates than places
    check_beam(beam(qa, x, score, None, 8, 5), x, score, None, 5)
    parent, token, out = beam(qa, x, score, None, 8, 5)
    assert (parent[1] == -1).all() and (token[1] == -1).all() and (out[1] == ninf).all()
    assert set(parent[3].tolist()) == {24} and sorted(zip(parent[4].tolist(), token[4].tolist()))[-3:] == [(33, 5), (36, 4), (36, 6)]


def test_beam_far_scores(qa, gpu):
    """a score that hides the others (-1e9): candidates of that beam only after all others"""
    x, _, _ = inputs(11, 4, 3, "f32")
    score = [-1.0, -1e9, -2.0, -1e9]
    parent, token, _ = beam(qa, x, score, None, 12, 1)
    assert set(parent[0, :6].tolist()) == {0, 2} and set(parent[0, 6:].tolist()) == {1, 3}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("beams,n_out,vocab", [(64, 64, 151936), (40, 64, 20000), (33, 48, 3000), (30, 30, 5000)])
def test_beam_more_candidates_than_a_list(qa, gpu, dtype, beams, n_out, vocab):
    """many beams and places: of thousands of shares nearly all may reach what the best ones do"""
    x, score, g = inputs(16, 2 * beams, vocab, dtype, 1.0)
    score = [-1.0 - 1e-3 * i for i in range(2 * beams)]
    ended = [i if i % 8 == 3 else -1 for i in range(2 * beams)]
    check_beam(beam(qa, x, score, ended, n_out, 2), x, score, ended, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("beams,n_out,vocab", [(4, 4, 151936), (12, 24, 30000), (40, 64, 20000), (64, 64, 5000)])
@pytest.mark.parametrize("kind", ["one far above", "far below", "near each other", "steps"])
def test_beam_ranges(qa, gpu, kind, dtype, beams, n_out, vocab):
    """what the candidates' range is cut by: one far above all others, nearly all far below, nearly all equal, few values"""
    x, score, g = inputs(17, beams, vocab, "f32", 1.0)
    if kind == "one far above":
        x[:, 7::5000] = 1e4
        x[beams // 2:, 7::5000] = 0.0
    elif kind == "far below":
        x[:, T.randperm(vocab, generator=g)[:vocab - n_out // 2].cuda()] -= 1e4
        score = [-1.0 if b % 3 else -5e4 for b in range(beams)]
    elif kind == "near each other":
        x = 5.0 + 1e-6 * x
    else:
        x = (x * 2).round() / 2
    x = x.to(DT[dtype])
    check_beam(beam(qa, x, score, None, n_out, 1), x, score, None, 1)


def test_beam_many_rows(qa, gpu):
    x, score, _ = inputs(12, 4096, 300)
    check_beam(beam(qa, x, score, None, 2, 512), x, score, None, 512)


def test_same_choice_every_time(qa, gpu):
    x, score, _ = inputs(13, 64, 151936, "bf16", 0.5)
    first = beam(qa, x, score, None, 16, 8)
    for _ in range(4):
        again = beam(qa, x, score, None, 16, 8)
        assert all((a == b).all() for a, b in zip(first, again))
    check_beam(first, x, score, None, 8)


def test_two_streams(qa, gpu):
    st = [T.cuda.Stream() for _ in range(2)]
    a, sa, _ = inputs(14, 8, 151936)
    b, sb, _ = inputs(15, 32, 20011)
    T.cuda.synchronize()
    L, keep = qa.lib(), []
    for x, s, seqs, n, stream in ((a, sa, 2, 4, st[0]), (b, sb, 4, 16, st[1])):
        need = L.qwen_hip_beam_select_ws_bytes(seqs, x.shape[0] // seqs, x.shape[1], n)
        keep.append((x, s, seqs, n, stream, T.empty(need, dtype=T.uint8, device="cuda"), T.tensor(s, device="cuda"),
                     T.zeros(2, seqs, n, dtype=T.int32, device="cuda"), T.zeros(seqs, n, device="cuda")))
    T.cuda.synchronize()
    for _ in range(5):
        for x, s, seqs, n, stream, ws, ds, ids, out in keep:
            qa.check(L.qwen_hip_beam_select(ids[0].data_ptr(), ids[1].data_ptr(), out.data_ptr(), x.data_ptr(), qa.ST_F32,
                                            x.shape[1], seqs, x.shape[0] // seqs, x.shape[1], ds.data_ptr(), None, n,
                                            ws.data_ptr(), ws.numel(), stream.cuda_stream))
    T.cuda.synchronize()
    for x, s, seqs, n, stream, ws, ds, ids, out in keep:
        check_beam((ids[0].cpu().numpy(), ids[1].cpu().numpy(), out.cpu().numpy()), x, s, None, seqs)

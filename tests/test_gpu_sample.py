"""qwen_hip_sample against its definition in 64 bits.  Tokens are whole numbers, so they have to be
equal; where a row's random number (or top_p's cut) falls within rounding of a border between two
tokens, either side is right.  Weights are off by at most 2^-22 of each (the exponential's 1 ulp and
its fraction's rounding to 24 bits, half a step each, and the cut at 2^-43 of the largest), so sums of
them and their ratios by 2^-21: borders are tried at u and top_p moved by that much."""
import math

import numpy as np
import pytest
import torch as T

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -21


def token(x, temp, k, p, least, u):
    """the definition, on one row of float64"""
    x = np.where(np.isnan(x), -np.inf, x)
    n = len(x)
    if not np.any(x > -np.inf):
        return -1
    order = np.argsort(-x, kind="stable")
    if not temp > 0:
        return int(order[0])
    m = x[order[0]]
    with np.errstate(invalid="ignore"):
        a = np.where(x == m, 0.0, (m - x) / temp)
    w = np.exp(-np.where(np.isnan(a), np.inf, a))
    order = order[x[order] > -np.inf]
    if 0 < k < n:
        order = order[:k]
    if not (math.isnan(p) or p >= 1):
        c = np.cumsum(w[order])
        before = np.concatenate([[0.0], c[:-1]])
        keep = before < max(p, 0.0) * c[-1]
        keep[0] = True
        order = order[keep]
    if least > 0:
        order = order[w[order] >= min(least, 1.0)]
    order = np.sort(order)
    c = np.cumsum(w[order])
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    return int(order[min(np.searchsorted(c, u * c[-1], side="right"), len(order) - 1)])


def allowed(x, temp, k, p, least, u):
    got = set()
    for dp in (0.0, -EPS, EPS):
        for du in (0.0, -EPS, EPS):
            # a cut at exactly 0 or 1 is no rounding matter
            got.add(token(x, temp, k, p + dp if 0 < p < 1 else p, least, u + du))
    return got


def draw(qa, x, temp=None, k=None, p=None, least=None, u=None, stride=None, stream=None):
    rows, vocab = x.shape
    stride = vocab if stride is None else stride
    buf = T.full((rows, stride), 1e30, dtype=T.float32)
    buf[:, :vocab] = x
    f = lambda v: None if v is None else T.tensor(v, dtype=T.float32).cuda()
    d = [buf.cuda(), f(temp), None if k is None else T.tensor(k, dtype=T.int32).cuda(), f(p), f(least), f(u)]
    ptr = [None if t is None else t.data_ptr() for t in d]
    need = qa.lib().qwen_hip_sample_ws_bytes(rows, vocab)
    ws = T.full((need,), 255, dtype=T.uint8, device="cuda")       # what it holds before does not matter
    out = T.full((rows,), -7, dtype=T.int32, device="cuda")
    T.cuda.synchronize()
    qa.check(qa.lib().qwen_hip_sample(out.data_ptr(), ptr[0], stride, rows, vocab, *ptr[1:], ws.data_ptr(), need,
                                      stream), "sample")
    T.cuda.synchronize()
    return out.cpu().tolist()


def check(qa, x, temp=None, k=None, p=None, least=None, u=None, stride=None):
    rows = x.shape[0]
    got = draw(qa, x, temp, k, p, least, u, stride)
    for r in range(rows):
        one = lambda v, off: off if v is None else np.float32(v[r]).item()
        ok = allowed(x[r].double().numpy(), one(temp, 1.0), 0 if k is None else k[r], one(p, 1.0), one(least, 0.0),
                     one(u, 0.0))
        assert got[r] in ok, (r, got[r], ok)
    return got


def logits(seed, rows, vocab, std):
    return T.randn(rows, vocab, generator=T.Generator().manual_seed(seed)) * std


def rnd(seed, rows, lo=0.0, hi=1.0):
    return (T.rand(rows, generator=T.Generator().manual_seed(seed)) * (hi - lo) + lo).tolist()


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 1024, 1025, 5000, 151936])
@pytest.mark.parametrize("mode", ["none", "k", "p", "min", "kp", "all"])
def test_modes(qa, gpu, vocab, mode):
    rows = 12
    x = logits(vocab, rows, vocab, 2.5)
    k = [1, 2, 5, 17, 40, 50, 64, 100, 300, vocab - 1, vocab, vocab + 5]
    check(qa, x, temp=rnd(1, rows, 0.5, 1.5), k=k if mode in ("k", "kp", "all") else None,
          p=rnd(2, rows) if mode in ("p", "kp", "all") else None,
          least=rnd(3, rows, 0.0, 0.3) if mode in ("min", "all") else None, u=rnd(4, rows))


@pytest.mark.parametrize("std", [0.01, 0.3, 1.0, 5.0, 30.0])
def test_spreads(qa, gpu, std):
    """from nearly equal logits (the thresholds' classes overflow the short list) to a few likely ones"""
    rows = 8
    check(qa, logits(7, rows, 151936, std), temp=[0.7] * rows, k=[0, 50, 1000, 0, 70000, 151000, 3, 0],
          p=[0.9, 0.5, 0.99, 0.1, 0.7, 0.999, 0.3, 1.0], u=rnd(8, rows))


@pytest.mark.parametrize("values", [1, 2, 7])
def test_ties(qa, gpu, values):
    """few different logits: thresholds inside runs of equal ones, which the lower index wins"""
    rows, vocab = 8, 20000
    g = T.Generator().manual_seed(9)
    x = T.randint(0, values, (rows, vocab), generator=g).float() * 0.25
    x[:, ::3] *= -1.0                       # zeros of both signs are equal
    check(qa, x, k=[1, 2, 500, 19999, 0, 0, 3000, 10000], p=[1.0, 1.0, 1.0, 1.0, 0.25, 0.75, 0.5, 1e-9],
          u=rnd(10, rows))
    check(qa, x, u=rnd(11, rows))


def test_edges_of_parameters(qa, gpu):
    nan, inf = math.nan, math.inf
    rows = 14
    x = logits(12, rows, 3001, 2.0)
    check(qa, x, temp=[0.0, -1.0, nan, inf, 1e-6, 1e6, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0],
          k=[5, 0, 0, 0, 0, 0, -3, 1, 0, 0, 0, 0, 0, 3001],
          p=[0.5, 1.0, 1.0, 1.0, 1.0, 0.5, 1.0, 1.0, 0.0, -1.0, nan, 1.5, 1.0, 1.0],
          least=[0.0, 0.0, 0.0, 0.0, 0.0, 0.0, nan, -1.0, 0.0, 0.0, 0.0, 0.0, 2.0, 1.0],
          u=[0.3, 0.999, 0.5, 0.5, 0.5, 0.5, 0.7, 0.99, 0.9, 0.9, 0.4, 0.6, 0.5, 0.9])
    # random numbers at and past the ends
    y = logits(13, 6, 500, 1.0)
    check(qa, y, u=[0.0, 1.0, -1.0, nan, 1 - 2.0 ** -24, 2.0])


def test_infinite_and_undefined_logits(qa, gpu):
    inf, nan = math.inf, math.nan
    x = logits(14, 8, 4000, 2.0)
    x[0] = -inf                              # nothing to draw
    x[1] = nan
    x[2, :3999] = -inf                       # one entry
    x[3, 100], x[3, 2000] = inf, inf         # two certain ones
    x[4, ::2] = nan
    x[5, 17] = inf
    x[6] = -3.4e38
    x[7, :2000] = -inf
    kw = dict(k=[5, 5, 5, 0, 50, 3, 0, 40], p=[0.9] * 8, u=rnd(15, 8))
    got = check(qa, x, **kw)
    assert got[0] == got[1] == -1 and got[2] == 3999 and got[3] in (100, 2000) and got[5] == 17
    assert check(qa, x, u=[0.4, 0.4, 0.4, 0.75, 0.4, 0.4, 0.4, 0.4])[3] == 2000


def test_all_of_them_and_rows_apart(qa, gpu):
    """defaults only; rows of a wider buffer whose other entries would win; many rows"""
    x = logits(16, 300, 777, 1.0)
    check(qa, x, u=rnd(17, 300), stride=801)
    check(qa, x[:, :1], u=rnd(18, 300))


def test_frequencies(qa, gpu):
    """u evenly over [0, 1) draws every kept entry as often as its share says (counted, not random)"""
    n = 4096
    x = T.log(T.tensor([[0.1, 0.4, 0.05, 0.25, 0.2]])).repeat(n, 1)
    got = np.bincount(draw(qa, x, u=[(i + 0.5) / n for i in range(n)]), minlength=5) / n
    assert np.all(np.abs(got - [0.1, 0.4, 0.05, 0.25, 0.2]) <= 1.0 / n)
    got = np.bincount(draw(qa, x, k=[3] * n, u=[(i + 0.5) / n for i in range(n)]), minlength=5) / n
    assert np.all(np.abs(got - np.array([0, 0.4, 0, 0.25, 0.2]) / 0.85) <= 1.0 / n)


def test_same_every_time(qa, gpu):
    x = logits(19, 32, 151936, 2.0)
    kw = dict(k=[0, 100] * 16, p=[0.95] * 32, u=rnd(20, 32))
    first = draw(qa, x, **kw)
    assert all(draw(qa, x, **kw) == first for _ in range(3))


def test_largest_sizes(qa, gpu):
    """the largest vocabulary, by the list and (nearly equal logits) by selection; the most rows"""
    vocab = 1 << 20
    kw = dict(k=[0, 50], p=[0.9, 0.99], u=rnd(21, 2))
    check(qa, logits(22, 2, vocab, 3.0), **kw)
    check(qa, logits(23, 2, vocab, 0.01), k=[0, 700000], p=[0.5, 0.8], u=rnd(24, 2))
    rows = 1 << 16
    x = logits(25, rows, 3, 1.0)
    got, u = draw(qa, x, u=rnd(26, rows)), rnd(26, rows)
    for r in list(range(0, rows, 997)) + [rows - 1]:
        assert got[r] in allowed(x[r].double().numpy(), 1.0, 0, 1.0, 0.0, np.float32(u[r]).item())
    assert set(got) == {0, 1, 2}


def test_two_streams(qa, gpu):
    """two draws that may overlap, a workspace and a stream each"""
    xs, us = [logits(27 + i, 16, 60000, 2.0) for i in range(2)], [rnd(29 + i, 16) for i in range(2)]
    p = [0.9] * 16
    want = [draw(qa, x, p=p, u=u) for x, u in zip(xs, us)]
    need = qa.lib().qwen_hip_sample_ws_bytes(16, 60000)
    d = [(x.cuda(), T.tensor(p).cuda(), T.tensor(u).cuda(), T.empty(need, dtype=T.uint8, device="cuda"),
          T.empty(16, dtype=T.int32, device="cuda"), T.cuda.Stream()) for x, u in zip(xs, us)]
    T.cuda.synchronize()
    for _ in range(5):
        for x, q, u, ws, out, st in d:
            qa.check(qa.lib().qwen_hip_sample(out.data_ptr(), x.data_ptr(), 60000, 16, 60000, None, None, q.data_ptr(),
                                              None, u.data_ptr(), ws.data_ptr(), need, st.cuda_stream))
    T.cuda.synchronize()
    assert [t[4].cpu().tolist() for t in d] == want

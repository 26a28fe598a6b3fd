"""How many bits the paged attention's operands keep on the matrix cores, which take bf16.  The cases are
made so that an operand held in too few terms shows: queries of one dim, whose scores are one
product each, and values whose weighted sum nearly cancels.  What a case must refuse is tried on the
CPU, with the terms' arithmetic written out here; the kernels are held to the same bounds."""
import math

import pytest
import torch as T

import paged_util as U
from paged_util import HD, Paged, check

E = 2.0 ** -24


def one_dim(seed, act, cache, group, lens, new=None, kv_heads=2):
    """queries of one dim each, of 1 to 2"""
    p = Paged(seed, lens, new=new, group=group, kv_heads=kv_heads, page=16, act=act, cache=cache)
    q = T.zeros(p.rows, p.heads, HD)
    at = T.randint(0, HD, (p.rows, p.heads, 1), generator=p.g)
    q.scatter_(2, at, 1.0 + T.rand(p.rows, p.heads, 1, generator=p.g))
    p.q = q.view(p.rows, -1).to(U.T[act])
    return p


def cancelling(p):
    """keys in pairs: elements of the second larger by a part in 128, the value the negative of the first"""
    for s, l in enumerate(p.lens):
        for i in range(1, l, 2):
            a, b = (p.page_of(s, i - 1), (i - 1) % p.page), (p.page_of(s, i), i % p.page)
            p.k[b[0], :, b[1]] = (p.k[a[0], :, a[1]].float() * (1 + 2.0 ** -7)).to(p.k.dtype)
            p.v[b[0], :, b[1]] = -p.v[a[0], :, a[1]]
    return p


def by_row(p):
    """(row, head, query, keys, values) in 64 bits of every row that sees something"""
    for s, (l, c) in enumerate(zip(p.lens, p.counts)):
        pid, slot = T.tensor([p.page_of(s, i) for i in range(l)]), T.arange(l) % p.page
        k, v = p.k[pid, :, slot].double(), p.v[pid, :, slot].double()
        for i in range(c):
            row, see = p.starts[s] + i, l - c + i + 1
            for h in range(p.heads):
                yield row, h, p.q[row].view(p.heads, HD)[h].double(), k[:see, h // p.group], v[:see, h // p.group]


def bounds(p, scale, roundings, weights=0.0):
    """(out, tolerance) as Paged.reference, but for a score of `roundings` half steps of fp32 (one
    product: its terms' sum and the scaling) and weights off by `weights` of each."""
    out = T.zeros(p.rows, p.heads, HD, dtype=T.float64)
    tol = T.zeros_like(out)
    for row, h, q, k, v in by_row(p):
        sc = k @ q * scale
        w, n = T.softmax(sc, 0), k.shape[0]
        off = roundings * E * (k.abs() @ q.abs() * scale) + 4 * E * (1 + sc.abs())
        rel = 2 * off.max() + 2 * (n + 8) * E + weights
        out[row, h] = w @ v
        tol[row, h] = 1.1 * (rel * (w @ v.abs()) + U.HALF[p.act] * (w @ v).abs()) + 1e-37
    return out.view(p.rows, -1), tol.view(p.rows, -1)


def held(x, n):
    """x in n bf16 terms, each rounded to nearest even"""
    got, left = T.zeros_like(x), x.float()
    for _ in range(n):
        t = left.bfloat16().float()
        got, left = got + t.double(), left - t
    return got


def emulate(p, scale, weights):
    """the attention with its weights in so many terms against exact values, rounded to the rows' type"""
    out = T.zeros(p.rows, p.heads, HD, dtype=T.float64)
    for row, h, q, k, v in by_row(p):
        sc = k @ q * scale
        x = T.exp(sc - sc.max())
        out[row, h] = (held(x, weights) @ v) / x.sum()
    return out.view(p.rows, -1).to(U.T[p.act])


def outside(got, want, tol):
    return int(((got.double().cpu() - want).abs() > tol).sum())


# ---------------------------------------------------------------------------
# bf16 rows: probabilities in two terms, fp32 values in two
# ---------------------------------------------------------------------------
WEIGHTS = {"bf16": 2.0 ** -16, "f32": 2.0 ** -14}
LENS = [2, 3, 16, 40, 300]


def bf16_rows(which, cache, group):
    new = None if which == "decode" else [2, 1, 16, 33, 70]
    return cancelling(one_dim(1 + group, "bf16", cache, group, LENS, new))


@pytest.mark.parametrize("which,cache,group", [("decode", "bf16", 8), ("prefill", "bf16", 2), ("prefill", "f32", 2)])
def test_bf16_rows_case_sees_one_term(which, cache, group):
    """probabilities of 8 bits are outside of the bound, of 16 inside"""
    p = bf16_rows(which, cache, group)
    want, tol = bounds(p, 1.0, 16, WEIGHTS[cache])
    assert outside(emulate(p, 1.0, 1), want, tol) > 0.1 * want.numel()
    assert outside(emulate(p, 1.0, 2), want, tol) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("cache", ["bf16", "f32"])
@pytest.mark.parametrize("group", [1, 2, 4, 5, 8, 16])
def test_bf16_rows_probabilities(qa, gpu, which, cache, group):
    """whatever the number of heads: an fp32 softmax, rounded once to the rows' type at the end"""
    p = bf16_rows(which, cache, group).gpu(qa)
    want, tol = bounds(p, 1.0, 16, WEIGHTS[cache])
    for max_len in (64, 300, 5000):                # both block shapes, split and unsplit
        check(p.attention(qa, 1.0, max_len=max_len), want, tol)


# ---------------------------------------------------------------------------
# what is no number, by any of its bits
# ---------------------------------------------------------------------------
NANS = [0x7f800001, 0x7f80ffff, 0xff800001 - (1 << 32), 0x7fc00000, 0x7fffffff, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("bits", NANS)
def test_undefined_values_by_any_bits(qa, gpu, which, act, bits):
    """a value of an fp32 cache is undefined whichever half of its word says so: the rows that see it are, and no
    others"""
    p = Paged(5, [70, 20], new=None if which == "decode" else [70, 20], group=2, kv_heads=2, page=16, act=act)
    for x, s, pos, h, d in ((p.v, 0, 40, 0, 3), (p.v, 0, 69, 1, 100), (p.k, 1, 10, 1, 64)):
        x.view(T.int32)[p.page_of(s, pos), h, pos % p.page, d] = bits
    p.gpu(qa)
    assert int(p.d["v"].view(T.int32)[p.page_of(0, 40), 0, 40 % p.page, 3]) == bits
    check(p.attention(qa, 1.0 / math.sqrt(HD)), *p.reference(1.0 / math.sqrt(HD)))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", NANS)
@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_append_undefined_by_any_bits(qa, gpu, cache, bits):
    """an undefined element of an fp32 row stays one in the pages"""
    import ctypes as C
    p = Paged(6, [3], group=1, kv_heads=1, page=4, cache=cache).gpu(qa)
    x = T.ones(1, 3 * HD)
    x.view(T.int32)[0, HD + 5] = x.view(T.int32)[0, 2 * HD + 6] = bits
    x, out = x.cuda(), T.zeros(1, HD, device="cuda")
    b = x.data_ptr()
    qa.check(qa.lib().qwen_hip_paged_append(C.byref(p.c_kv), C.byref(p.c_batch), out.data_ptr(), b, b + 4 * HD,
                                            b + 8 * HD, p.c_act, HD, HD, 1, None, None, 0.0, None, None, 0, None))
    T.cuda.synchronize()
    i = p.page_of(0, 2)
    k, v = p.d["k"][i, 0, 2].float().cpu(), p.d["v"][i, 0, 2].float().cpu()
    assert T.isnan(k).nonzero().tolist() == [[5]] and T.isnan(v).nonzero().tolist() == [[6]]


# ---------------------------------------------------------------------------
# fp32 rows: every operand in three terms, whose products lose 2^-24 at most
# ---------------------------------------------------------------------------
# Half steps of fp32 that a score of one product may be off by: one for the dropped terms, one step
# of the sum that adds the largest term, and those of the sums before it, a part in 256 of it.
ONE_PRODUCT = 3.5


def first_order(p, scale, roundings):
    """(out, tolerance) to first order in the scores' errors: d out = sum w_j (v_j - out) d s_j.  A
    score is off by `roundings` half steps of itself (none where the key's element is a power of two:
    then its product is the query's terms moved), and, as the difference to the largest that the
    exponential takes, by 6 of 1 + |difference| (the scaling's two roundings, which all keys of a
    query of one dim share, the difference's own, the exponential's ulp and its argument); the
    sums over n keys by n + 8 half steps of their absolute terms each."""
    out = T.zeros(p.rows, p.heads, HD, dtype=T.float64)
    tol = T.zeros_like(out)
    for row, h, q, k, v in by_row(p):
        sc = k @ q * scale
        w, n = T.softmax(sc, 0), k.shape[0]
        o = w @ v
        moved = T.frexp(k[:, int(q.abs().argmax())])[0].abs() == 0.5
        off = T.where(moved, 0.0, roundings * E * sc.abs()) + 6 * E * (1 + (sc - sc.max()).abs())
        out[row, h] = o
        tol[row, h] = 1.1 * ((w * off) @ (v - o).abs() + 2 * (n + 8) * E * (w @ v.abs()) + U.HALF[p.act] * o.abs()) + 1e-37
    return out.view(p.rows, -1), tol.view(p.rows, -1)


def parts(x, n, cut=False):
    """n bf16 terms of fp32 values, each rounded to nearest even or cut off"""
    got, left, most = [], x.float(), T.finfo(T.bfloat16).max
    for _ in range(n):
        t = (left.view(T.int32) & -65536).view(T.float32) if cut else left.clamp(-most, most).bfloat16().float()
        got.append(t.double())
        left = left - t
    return got


def emulate_terms(p, scale, n=3, cut=False, which="qkpv"):
    """the attention with the products of n terms (pairs i + j < n) of the operands in `which` against exact values"""
    def times(a, b, product, names):
        if not all(x in which for x in names):
            return product(a, b)
        return sum(product(x, y) for i, x in enumerate(parts(a, n, cut)) for j, y in enumerate(parts(b, n, cut)) if i + j < n)

    out = T.zeros(p.rows, p.heads, HD, dtype=T.float64)
    for row, h, q, k, v in by_row(p):
        sc = times(k, q, lambda a, b: a @ b, "qk") * scale
        x = T.exp(sc - sc.max()).float().double()
        out[row, h] = times(x, v, lambda a, b: a @ b, "pv") / x.sum()
    return out.view(p.rows, -1)


F32_LENS = [2, 2, 3, 4, 9, 33]


def wide(which, cache, group):
    """scores some units apart, all of their bits in use"""
    p = one_dim(20 + group, "f32", cache, group, F32_LENS * 4, None if which == "decode" else [2, 1, 3, 2, 5, 20] * 4)
    p.k = (2 * p.k.float()).to(p.k.dtype)
    return p, 1.0


def near(which, cache, group):
    """scores of hundreds within a few units: queries and every other key a little below 1 + 2^-7, where terms
    that are cut off leave the most behind, the other keys 1"""
    p = one_dim(40 + group, "f32", cache, group, F32_LENS * 4, None if which == "decode" else [2, 1, 3, 2, 5, 20] * 4)
    low = lambda *s: 1 + 2.0 ** -7 - T.randint(1, 100, s, generator=p.g).double() * 2.0 ** -23
    p.q = T.where(p.q == 0, 0.0, 512 * low(*p.q.shape)).float()
    k = low(*p.k.shape)
    k[:, :, ::2] = 1.0
    p.k = T.where(T.isnan(p.k.double()), math.nan, k).to(p.k.dtype)
    return p, math.log(2.0)


def weights(which, cache, group):
    """two keys whose scores are exact, one value of 1 and one of 0: the weight itself"""
    n = 96
    p = Paged(60 + group, [2] * n, new=None if which == "decode" else [1] * n, group=group, kv_heads=1, page=4, cache=cache)
    p.q = T.zeros(n, p.heads, HD)
    p.q[..., 7] = 1.0
    p.q = p.q.view(n, -1)
    for s in range(n):
        i = p.page_of(s, 0)
        p.k[i, :, :2, 7] = T.randint(-24, 25, (1, 2), generator=p.g).to(p.k.dtype) / 16
        p.v[i, :, 0], p.v[i, :, 1] = 1.0, 0.0
    return p, 1.0


CASES = [(wide, "f32", "qk"), (wide, "bf16", "qk"), (weights, "f32", "pv"), (weights, "bf16", "pv"), (near, "f32", "qk")]


@pytest.mark.parametrize("make,cache,operands", CASES[:-1])
def test_f32_rows_case_sees_two_terms(make, cache, operands):
    """operands in two terms are outside of the bound, in three (to nearest) inside"""
    p, scale = make("prefill", cache, 8)
    want, tol = first_order(p, scale, ONE_PRODUCT)
    assert outside(emulate_terms(p, scale, 2, which=operands), want, tol) > 0.005 * want.numel()
    assert outside(emulate_terms(p, scale), want, tol) == 0


def test_f32_rows_case_sees_terms_cut_off():
    """three terms that are cut off, not rounded, lose up to 2^-21 of a product"""
    p, scale = near("prefill", "f32", 8)
    want, tol = first_order(p, scale, ONE_PRODUCT)
    assert outside(emulate_terms(p, scale, cut=True, which="qk"), want, tol) > 0.02 * want.numel()


def test_products_of_three_terms():
    """what the pairs i + j <= 2 drop: below 2^-24 of the product to nearest, up to 2^-21 cut off"""
    g = T.Generator().manual_seed(9)
    x, y = ((1 + T.rand(1 << 20, generator=g)).float() for _ in range(2))
    x[:4096], y[:4096] = 1 + 2.0 ** -7 - T.rand(4096, generator=g) * 2.0 ** -16, 1 + 2.0 ** -7 - T.rand(4096, generator=g) * 2.0 ** -16
    x[4096:8192], y[4096:8192] = 1 + 2.0 ** -8 - T.rand(4096, generator=g) * 2.0 ** -15, 1 + 2.0 ** -8 - T.rand(4096, generator=g) * 2.0 ** -15
    loss = lambda cut: float(((sum(a * b for i, a in enumerate(parts(x, 3, cut)) for j, b in enumerate(parts(y, 3, cut))
                                   if i + j <= 2)) / (x.double() * y.double()) - 1).abs().max())
    assert loss(False) <= 2.0 ** -24 < 4 * 2.0 ** -24 < loss(True) < 2.0 ** -21
    for z in (x, y, T.tensor([3.4e38, -3.39e38, 1e-30])):
        assert T.equal(sum(parts(z, 3, False)), z.double())     # three terms are the value


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("group", [1, 2, 4, 8])
@pytest.mark.parametrize("make,cache,operands", CASES)
def test_f32_rows_terms(qa, gpu, make, cache, operands, group, which):
    p, scale = make(which, cache, group)
    p.gpu(qa)
    want, tol = first_order(p, scale, ONE_PRODUCT)
    for max_len in (33, 300, 5000):
        check(p.attention(qa, scale, max_len=max_len), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 8])
def test_f32_rows_one_key(qa, gpu, which, cache, group):
    """a row that sees one key gets its value, bit for bit: the largest numbers, which round to an infinity as
    bf16, among them"""
    p = Paged(80 + group, [1] * 40, new=None if which == "decode" else [1] * 40, group=group, kv_heads=2, page=16, cache=cache)
    big = T.finfo(T.float32).max if cache == "f32" else T.finfo(T.bfloat16).max
    for s in range(0, 40, 3):
        p.v[p.page_of(s, 0), :, 0, 11], p.v[p.page_of(s, 0), :, 0, 90] = big, -big * (1 - 2.0 ** -10)
    p.gpu(qa)
    want = T.stack([p.v[p.page_of(s, 0), :, 0].float().repeat_interleave(group, 0).flatten() for s in range(40)])
    for max_len in (1, 300, 5000):
        assert T.equal(p.attention(qa, 1.0, max_len=max_len).cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_f32_largest_numbers(qa, gpu, which):
    """queries and keys that round to an infinity as bf16"""
    p = Paged(90, [2, 2], new=None if which == "decode" else [1, 1], group=2, kv_heads=1, page=16)
    big = T.finfo(T.float32).max
    p.q.zero_()
    p.q[0, [5, HD + 5]], p.q[1, [5, HD + 5]] = T.tensor([big, -big]), T.tensor([2.0 ** -126, -2.0 ** -126])
    i, j = p.page_of(0, 0), p.page_of(1, 0)
    p.k[i, 0, :2], p.k[j, 0, :2] = 0.0, 0.0
    p.k[i, 0, 0, 5], p.k[i, 0, 1, 5] = 2.0 ** -126, 2.0 ** -125
    p.k[j, 0, 0, 5], p.k[j, 0, 1, 5] = big, -big
    check(p.gpu(qa).attention(qa, math.log(2.0)), *first_order(p, math.log(2.0), ONE_PRODUCT))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_nearly_even_weights(qa, gpu, which, cache):
    p = Paged(34, [257, 64], new=None if which == "decode" else [40, 64], group=8, kv_heads=2, page=16, cache=cache)
    check(p.gpu(qa).attention(qa, 1e-3), *p.reference(1e-3))

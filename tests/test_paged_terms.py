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
# bf16 rows: probabilities in two terms (2^-17 of each), fp32 values in two (2^-15)
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

"""The paged cache's operators through the C ABI on device memory, against their definitions in 64
bits (tests/paged_util.py, which also derives the tolerances): appending normed and rotated rows,
attention of single tokens and of packed prompts."""
import ctypes as C
import math

import pytest
import torch as T

import paged_util as U
from paged_util import HD, Paged, check

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(HD)
TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")]


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def run_append(qa, p, norm=True, rope=True, n_pos=None, pad=0, in_place=False, stream=None):
    """(q_out, k pages, v pages) of the library and of the definition, and their tolerances"""
    g, H, KH = p.g, p.heads, p.kv_heads
    dt = U.T[p.act]
    width = (H + 2 * KH) * HD + pad
    wide = T.randn(p.rows, width, generator=g).to(dt)          # one row: q | k | v | pad
    if in_place:
        q, qs = T.randn(p.rows, H * HD, generator=g).to(dt), H * HD
    else:
        q, qs = wide[:, :H * HD], width
    k, v = wide[:, H * HD:(H + KH) * HD], wide[:, (H + KH) * HD:(H + 2 * KH) * HD]
    wq, wk = (1 + 0.1 * T.randn(HD, generator=g) for _ in range(2))
    n_pos = max(p.lens + [1]) if n_pos is None else n_pos
    cos, sin = U.rope_tables(n_pos)
    d = [x.cuda() for x in (wide, wq, wk, cos, sin, q.contiguous())]
    size = wide.element_size()
    base = d[0].data_ptr()
    pq = d[5].data_ptr() if in_place else base
    out = d[5] if in_place else T.full((p.rows, H * HD), 7.0, dtype=dt, device="cuda")
    T.cuda.synchronize()
    rc = qa.lib().qwen_hip_paged_append(
        C.byref(p.c_kv), C.byref(p.c_batch), out.data_ptr(), pq, base + size * H * HD, base + size * (H + KH) * HD,
        p.c_act, qs, width, H, d[1].data_ptr() if norm else None, d[2].data_ptr() if norm else None, 1e-6,
        d[3].data_ptr() if rope else None, d[4].data_ptr() if rope else None, n_pos, stream)
    qa.check(rc, "append")
    T.cuda.synchronize()

    want_q = q.double().clone() if in_place else T.full((p.rows, H * HD), 7.0, dtype=T.float64)
    want_k, want_v = p.k.double().clone(), p.v.double().clone()
    tol_q, tol_k = T.zeros_like(want_q), T.zeros_like(want_k)
    # the norm: 8 products a lane and 4 sums over lanes, mean, reciprocal root (1 ulp): under 16
    # roundings of the scale; two products with the weight and the scale; the rotation's product,
    # fma: two of |a c| + |b s|.  20 half steps of fp32 of the terms' absolute sum, then the type's
    e = 20 * 2.0 ** -24
    for s, (l, c) in enumerate(zip(p.lens, p.counts)):
        for i in range(c):
            row, pos = p.starts[s] + i, max(l, 0) - c + i
            if pos < 0 or pos >= p.table.shape[1] * p.page or (rope and pos >= n_pos):
                continue
            cs, sn = (cos[pos], sin[pos]) if rope else (None, None)
            def both(x, w):
                y = U.norm_rope(x, w if norm else None, 1e-6, cs, sn)
                a = U.norm_rope(x.double().abs(), w.abs() if norm else None, 1e-6,
                                cs.abs() if rope else None, -sn.abs() if rope else None)
                lo = U.norm_rope(x.double().abs(), w.abs() if norm else None, 1e-6,
                                 cs.abs() if rope else None, sn.abs() if rope else None)
                return y, T.maximum(a, lo)      # both halves of |a c| + |b s|
            y, a = both(q[row].view(H, HD), wq)
            want_q[row], tol_q[row] = y.flatten(), (e * a + U.HALF[p.act] * y.abs()).flatten() + 1e-37
            pid = p.page_of(s, pos)
            if pid >= 0:
                y, a = both(k[row].view(KH, HD), wk)
                want_k[pid, :, pos % p.page] = y
                tol_k[pid, :, pos % p.page] = e * a + U.HALF[p.cache] * y.abs() + 1e-37
                want_v[pid, :, pos % p.page] = v[row].view(KH, HD).to(U.T[p.cache]).double()
    return (out.cpu(), p.d["k"].cpu(), p.d["v"].cpu()), (want_q, want_k, want_v), (tol_q, tol_k, T.zeros_like(want_v))


def check_append(got, want, tol):
    for n, g, w, t in zip("qkv", got, want, tol):
        g = g.double()
        same_nan = T.isnan(g) & T.isnan(w)
        bad = ~same_nan & ~((g - w).abs() <= t)
        assert not bool(bad.any()), (n, int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False), (False, False)])
def test_append_packed(qa, gpu, act, cache, norm, rope):
    """prompts of different lengths behind cached pasts, a sequence without rows, rows of no sequence
    before and behind, rows of a wider buffer"""
    p = Paged(1, [5, 40, 16, 33], new=[5, 7, 0, 33], group=3, kv_heads=2, page=8, act=act, cache=cache, front=2,
              back=3).gpu(qa)
    check_append(*run_append(qa, p, norm, rope, pad=8))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("group,kv_heads,page", [(1, 1, 1), (2, 8, 16), (8, 1, 256), (5, 3, 2)])
def test_append_token(qa, gpu, act, cache, group, kv_heads, page):
    """one row per sequence, the first slot of a page and the last among them"""
    p = Paged(2, [1, page, page + 1, 3 * page - 1 or 1, 70], group=group, kv_heads=kv_heads, page=page, act=act,
              cache=cache).gpu(qa)
    check_append(*run_append(qa, p))


def test_append_many_sequences(qa, gpu):
    """more sequences than one search step has lanes, some without rows"""
    lens = [(7 * i) % 23 + 1 for i in range(300)]
    p = Paged(3, lens, new=[min(l, i % 4) for i, l in enumerate(lens)], group=2, kv_heads=1, page=4, front=1, back=1)
    check_append(*run_append(qa, p.gpu(qa)))


def test_append_left_out(qa, gpu):
    """nothing is written for negative positions, positions past the rotation's table or the page table;
    a row whose page id is none of the cache's gets its query and stores nothing"""
    p = Paged(4, [3, 0, 20, 12, -2], new=[6, 2, 9, 4, 1], group=2, kv_heads=2, page=4)
    p.table[3, 2] = p.n_pages           # position 8 .. 11: an id one past the last page
    p.table[2, 3] = -1                  # position 12 .. 15 of sequence 2
    p.table[2, 4] = -2 ** 31
    p.gpu(qa)
    check_append(*run_append(qa, p, n_pos=18))
    q = Paged(5, [60], new=[60], group=2, kv_heads=1, page=4)
    q.table = q.table[:, :10].contiguous()     # a table of 40 positions
    check_append(*run_append(qa, q.gpu(qa)))


def test_append_in_place(qa, gpu):
    p = Paged(6, [9, 4], new=[4, 4], group=4, kv_heads=2, page=16, act="bf16", cache="bf16", back=2).gpu(qa)
    check_append(*run_append(qa, p, in_place=True))


def test_append_infinite_rows(qa, gpu):
    """without a norm and rotation keys and values go through as they are, infinite or none"""
    p = Paged(7, [4], group=1, kv_heads=1, page=4).gpu(qa)
    x = T.zeros(1, 3 * HD, device="cuda")
    x[0, HD], x[0, HD + 1], x[0, 2 * HD] = math.inf, math.nan, -math.inf
    out = T.zeros(1, HD, device="cuda")
    b = x.data_ptr()
    qa.check(qa.lib().qwen_hip_paged_append(C.byref(p.c_kv), C.byref(p.c_batch), out.data_ptr(), b, b + 4 * HD,
                                            b + 8 * HD, p.c_act, HD, HD, 1, None, None, 0.0, None, None, 0, None))
    T.cuda.synchronize()
    i = p.page_of(0, 3)
    assert float(p.d["k"][i, 0, 3, 0]) == math.inf and math.isnan(float(p.d["k"][i, 0, 3, 1]))
    assert float(p.d["v"][i, 0, 3, 0]) == -math.inf and float(p.d["v"][i, 0, 3, 1]) == 0.0


# ---------------------------------------------------------------------------
# attention of single tokens
# ---------------------------------------------------------------------------
LENS = [0, 1, 15, 16, 17, 63, 64, 65, 200, 530]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9, 16])
def test_decode_groups(qa, gpu, act, cache, group):
    p = Paged(10 + group, LENS, group=group, kv_heads=2, page=16, act=act, cache=cache).gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("page", [1, 2, 8, 64, 512])
@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_decode_pages(qa, gpu, page, cache):
    p = Paged(30, LENS, group=2, kv_heads=3, page=page, cache=cache).gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("max_len", [0, 1, 64, 100, 2 ** 31 - 1])
def test_any_max_len(qa, gpu, which, max_len):
    """max_len shapes the launch; results hold whatever it says"""
    p = Paged(31, [1, 900, 130, 0], new=None if which == "decode" else [1, 3, 130, 0], group=2, kv_heads=2, page=32)
    check(p.gpu(qa).attention(qa, SCALE, max_len=max_len), *p.reference(SCALE))


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("act,cache", TYPES)
def test_missing_pages(qa, gpu, which, act, cache):
    """positions whose page id is outside the cache are not there: a window that has let its first
    pages go, ids one past the end, the lowest number, a sequence without any page"""
    p = Paged(32, [300, 100, 64, 40], new=None if which == "decode" else [5, 100, 64, 2], group=2, kv_heads=2,
              page=16, act=act, cache=cache)
    p.table[0, :10] = -1
    p.table[1, 3] = p.n_pages
    p.table[1, 5] = 2 ** 31 - 1
    p.table[2, :] = -2 ** 31
    p.table[3, 1] = -5
    check(p.gpu(qa).attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_longer_than_the_table(qa, gpu, which):
    """a length past the page table's end: the positions that it holds are seen"""
    p = Paged(33, [100, 20], new=None if which == "decode" else [30, 20], group=2, kv_heads=1, page=8)
    p.table = p.table[:, :6].contiguous()
    check(p.gpu(qa).attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 8.0])
def test_scales(qa, gpu, which, scale):
    """nearly even weights, and scores of hundreds where one key takes all"""
    p = Paged(34, [257, 64], new=None if which == "decode" else [40, 64], group=2, kv_heads=2, page=16)
    check(p.gpu(qa).attention(qa, scale), *p.reference(scale))


def test_decode_infinite_values(qa, gpu):
    """an infinite or undefined value that a row sees reaches its outputs and no others"""
    p = Paged(35, [70, 70, 70], group=2, kv_heads=2, page=16)
    p.v[p.page_of(1, 20), 0, 20 % 16, 5] = math.inf
    p.v[p.page_of(1, 60), 1, 60 % 16, 9] = math.nan
    p.k[p.page_of(2, 3), 1, 3, 0] = math.nan
    check(p.gpu(qa).attention(qa, SCALE), *p.reference(SCALE))


# ---------------------------------------------------------------------------
# attention of packed prompts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("group,kv_heads", [(1, 2), (2, 2), (3, 1), (8, 1), (16, 1)])
def test_prefill_packed(qa, gpu, act, cache, group, kv_heads):
    """prompts from one row to several tiles, behind pasts, with a sequence without rows between and rows
    of no sequence around"""
    p = Paged(40 + group, [1, 70, 33, 90, 64, 150], new=[1, 70, 0, 31, 2, 97], group=group, kv_heads=kv_heads, page=16,
              act=act, cache=cache, front=3, back=5).gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("page", [1, 4, 128])
def test_prefill_pages(qa, gpu, act, cache, page):
    p = Paged(60, [31, 32, 33, 5], new=[31, 32, 33, 5], group=2, kv_heads=2, page=page, act=act, cache=cache).gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,cache", TYPES)
def test_prefill_chunk_split(qa, gpu, act, cache):
    """a few rows behind a long past: the keys are split over blocks"""
    p = Paged(61, [1024, 700], new=[31, 2], group=2, kv_heads=2, page=16, act=act, cache=cache).gpu(qa)
    assert qa.lib().qwen_hip_paged_attention_ws_bytes(C.byref(p.c_kv), C.byref(p.c_batch), p.heads) > 0
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,cache", TYPES)
def test_prefill_unsplit(qa, gpu, act, cache):
    """enough rows that no split is planned (max_len one tile)"""
    p = Paged(62, [300, 200], new=[300, 180], group=2, kv_heads=1, page=64, act=act, cache=cache).gpu(qa)
    check(p.attention(qa, SCALE, max_len=64), *p.reference(SCALE))


def test_prefill_more_rows_than_positions(qa, gpu):
    """rows at negative positions see nothing: zeros"""
    p = Paged(63, [3, 0, -4, 40], new=[5, 4, 2, 40], group=2, kv_heads=2, page=8, back=1).gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


def test_prefill_many_sequences(qa, gpu):
    lens = [(5 * i) % 11 + 1 for i in range(200)]
    p = Paged(64, lens, new=[min(l, i % 3) for i, l in enumerate(lens)], group=2, kv_heads=1, page=4, front=2).gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("split", [False, True])
def test_prefill_infinite_values(qa, gpu, act, cache, split):
    """infinite and undefined keys and values at positions that earlier rows of the same tile do not
    see: those rows keep their finite results, later ones get what the formula says"""
    p = Paged(65, [90, 70], new=[90, 70], group=2, kv_heads=2, page=16, act=act, cache=cache)
    def at(x, s, pos, h, d, v):
        x[p.page_of(s, pos), h, pos % p.page, d] = v
    at(p.v, 0, 20, 0, 3, math.inf)
    at(p.v, 0, 50, 0, 3, -math.inf)          # with the other: undefined from row 50 on
    at(p.v, 0, 40, 1, 7, -math.inf)
    at(p.v, 0, 80, 1, 100, math.nan)
    at(p.k, 1, 33, 0, 0, math.nan)
    at(p.v, 1, 0, 1, 127, math.inf)          # seen by every row
    check(p.gpu(qa).attention(qa, SCALE, max_len=None if split else 32), *p.reference(SCALE))


def test_prefill_is_decode_for_one_row(qa, gpu):
    """one row per sequence through either entry point, within both tolerances"""
    a = Paged(66, LENS[1:], group=2, kv_heads=2, page=16).gpu(qa)
    b = Paged(66, LENS[1:], new=[1] * len(LENS[1:]), group=2, kv_heads=2, page=16).gpu(qa)
    x, y = a.attention(qa, SCALE).double(), b.attention(qa, SCALE).double()
    tol = a.reference(SCALE)[1]
    assert bool(((x - y).abs().cpu() <= 2 * tol).all())


# ---------------------------------------------------------------------------
# memory, streams, graphs
# ---------------------------------------------------------------------------
def test_past_32_bit_offsets(qa, gpu):
    """a cache of more than 2^32 values: append to its last page and read it back"""
    page, KH = 4096, 8
    n_pages = (1 << 32) // (page * KH * HD) + 2
    k = T.empty(n_pages, KH, page, HD, dtype=T.bfloat16, device="cuda")
    v = T.empty_like(k)
    table = T.tensor([[n_pages - 1]], dtype=T.int32, device="cuda")
    lens = T.tensor([3], dtype=T.int32, device="cuda")
    start = T.tensor([0, 3], dtype=T.int32, device="cuda")
    g = T.Generator().manual_seed(5)
    x = T.randn(3, (16 + 16) * HD, generator=g).bfloat16().cuda()
    q = T.empty(3, 16 * HD, dtype=T.bfloat16, device="cuda")
    ckv = qa.PagedKV(k.data_ptr(), v.data_ptr(), table.data_ptr(), qa.ST_BF16, n_pages, page, KH, HD, 1, 1)
    cb = qa.PagedBatch(start.data_ptr(), lens.data_ptr(), 3, 3)
    L, b, w = qa.lib(), x.data_ptr(), 32 * HD
    qa.check(L.qwen_hip_paged_append(C.byref(ckv), C.byref(cb), q.data_ptr(), b, b + 2 * 16 * HD, b + 2 * 24 * HD,
                                     qa.ST_BF16, w, w, 16, None, None, 0.0, None, None, 0, None))
    T.cuda.synchronize()
    assert T.equal(k[-1, :, :3].transpose(0, 1).reshape(3, -1), x[:, 16 * HD:24 * HD])
    assert T.equal(v[-1, :, :3].transpose(0, 1).reshape(3, -1), x[:, 24 * HD:])
    p = Paged(0, [3], new=[3], group=2, kv_heads=KH, page=4, act="bf16", cache="bf16", spare=0)
    p.q = x[:, :16 * HD].cpu()
    kk, vv = x[:, 16 * HD:24 * HD].cpu().view(3, KH, HD), x[:, 24 * HD:].cpu().view(3, KH, HD)
    p.k[p.page_of(0, 0), :, :3], p.v[p.page_of(0, 0), :, :3] = kk.transpose(0, 1), vv.transpose(0, 1)
    want, tol = p.reference(SCALE)
    need = L.qwen_hip_paged_attention_ws_bytes(C.byref(ckv), C.byref(cb), 16)
    ws = T.empty(max(need, 16), dtype=T.uint8, device="cuda")
    out = T.empty_like(q)
    qa.check(L.qwen_hip_paged_attention_prefill(C.byref(ckv), C.byref(cb), out.data_ptr(), q.data_ptr(), qa.ST_BF16,
                                                16, SCALE, ws.data_ptr(), need, None))
    T.cuda.synchronize()
    check(out, want, tol)
    one = qa.PagedBatch(None, lens.data_ptr(), 1, 0)
    need = L.qwen_hip_paged_attention_ws_bytes(C.byref(ckv), C.byref(one), 16)
    ws = T.empty(max(need, 16), dtype=T.uint8, device="cuda")
    qa.check(L.qwen_hip_paged_attention_decode(C.byref(ckv), C.byref(one), out.data_ptr(), q[2:].contiguous().data_ptr(),
                                               qa.ST_BF16, 16, SCALE, ws.data_ptr(), need, None))
    T.cuda.synchronize()
    check(out[:1], want[2:], tol[2:])


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_past_32_bits_in_a_page(qa, gpu, which):
    """one page of 2^24 positions, the sequence ending where a slot's byte offset has passed 2^32.  Keys
    and values are 0 but for the last 40 positions, whose scores are near 200: what is before them
    weighs e^-200 each, so the answer is theirs alone."""
    page, length, n = 1 << 24, (1 << 23) + 77, 3 if which == "prefill" else 1
    g = T.Generator().manual_seed(8)
    k, v = (T.zeros(1, 1, page, HD, device="cuda") for _ in range(2))
    q = T.randn(1, HD, generator=g).repeat(n, 1)
    kk = q[:1] * (200 / SCALE / float((q[0] * q[0]).sum())) + 0.05 * T.randn(40, HD, generator=g)
    vv = T.randn(40, HD, generator=g)
    k[0, 0, length - 40:length], v[0, 0, length - 40:length] = kk.cuda(), vv.cuda()
    table, lens = T.zeros(1, 1, dtype=T.int32, device="cuda"), T.tensor([length], dtype=T.int32, device="cuda")
    start = T.tensor([0, n], dtype=T.int32, device="cuda")
    kv = qa.PagedKV(k.data_ptr(), v.data_ptr(), table.data_ptr(), qa.ST_F32, 1, page, 1, HD, 1, 1)
    b = qa.PagedBatch(start.data_ptr() if which == "prefill" else None, lens.data_ptr(), n, length)
    L, by = qa.lib(), (C.byref(kv), C.byref(b))
    need = L.qwen_hip_paged_attention_ws_bytes(*by, 1)
    ws, dq = T.empty(max(need, 16), dtype=T.uint8, device="cuda"), q.cuda()
    out = T.empty_like(dq)
    call = getattr(L, "qwen_hip_paged_attention_" + which)
    qa.check(call(*by, out.data_ptr(), dq.data_ptr(), qa.ST_F32, 1, SCALE, ws.data_ptr(), need, None))
    T.cuda.synchronize()
    for i in range(n):
        see = 40 - (n - 1 - i)
        x, y, z = kk[:see].double(), vv[:see].double(), q[i].double()
        sc = x @ z * SCALE
        w, e = T.softmax(sc, 0), 2.0 ** -24
        # paged_util's bound; weights of 0 add nothing to the sums, which join 64 splits at most
        rel = 2 * (136 * e * (x.abs() @ z.abs() * SCALE) + 4 * e * (1 + sc.abs())).max() + 2 * (see + 64 + 8) * e
        assert bool(((out[i].cpu().double() - w @ y).abs() <= 1.1 * (rel * (w @ y.abs()) + e * (w @ y).abs())).all())


def test_two_streams(qa, gpu):
    """two calls that may overlap, on streams of their own with a workspace each"""
    ps = [Paged(70 + i, [900, 33, 500], group=2, kv_heads=2, page=16).gpu(qa) for i in range(2)]
    streams = [T.cuda.Stream() for _ in ps]
    T.cuda.synchronize()
    outs, keep = [], []
    for p, st in zip(ps, streams):
        by = C.byref(p.c_kv), C.byref(p.c_batch)
        need = qa.lib().qwen_hip_paged_attention_ws_bytes(*by, p.heads)
        ws = T.empty(need, dtype=T.uint8, device="cuda")
        out = T.empty_like(p.d["q"])
        T.cuda.synchronize()
        for _ in range(5):
            qa.check(qa.lib().qwen_hip_paged_attention_decode(*by, out.data_ptr(), p.d["q"].data_ptr(), p.c_act,
                                                              p.heads, SCALE, ws.data_ptr(), need, st.cuda_stream))
        outs.append(out)
        keep.append(ws)
    T.cuda.synchronize()
    for p, out in zip(ps, outs):
        check(out, *p.reference(SCALE))


def test_same_bits_every_time(qa, gpu):
    for new in (None, [40, 33, 500]):
        p = Paged(72, [900, 33, 500], new=new, group=2, kv_heads=2, page=16).gpu(qa)
        first = p.attention(qa, SCALE)
        for _ in range(3):
            assert T.equal(first, p.attention(qa, SCALE))


# ---------------------------------------------------------------------------
# single tokens of many heads a kv head on a bf16 cache: the matrix cores' kernel
# ---------------------------------------------------------------------------
MANY = [("bf16", 8), ("f32", 12)]


@pytest.mark.parametrize("page", [1, 4, 64, 512])
@pytest.mark.parametrize("act,group", MANY)
def test_many_heads_pages(qa, gpu, act, group, page):
    p = Paged(60, LENS, group=group, kv_heads=1, page=page, act=act, cache="bf16").gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,group", MANY)
def test_many_heads_many_sequences(qa, gpu, act, group):
    lens = [(5 * i) % 40 for i in range(150)]
    p = Paged(61, lens, group=group, kv_heads=2, page=16, act=act, cache="bf16").gpu(qa)
    check(p.attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,group", MANY)
def test_many_heads_missing_pages_and_infinite_values(qa, gpu, act, group):
    p = Paged(62, [300, 100, 64, 70], group=group, kv_heads=2, page=16, act=act, cache="bf16")
    p.table[0, :10] = -1
    p.table[1, 3] = p.n_pages
    p.table[2, :] = -2 ** 31
    p.v[p.page_of(3, 20), 0, 20 % 16, 5] = math.inf
    p.v[p.page_of(3, 60), 1, 60 % 16, 9] = math.nan
    check(p.gpu(qa).attention(qa, SCALE), *p.reference(SCALE))


@pytest.mark.parametrize("act,group", MANY)
def test_many_heads_any_max_len(qa, gpu, act, group):
    p = Paged(63, [1, 900, 130, 0], group=group, kv_heads=1, page=32, act=act, cache="bf16").gpu(qa)
    for max_len in (0, 1, 100, 2 ** 31 - 1):
        check(p.attention(qa, SCALE, max_len=max_len), *p.reference(SCALE))


# ---------------------------------------------------------------------------
# prompts: both block shapes (max_len decides), and walks longer than 64 tiles
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("max_len", [64, 700, 900, 5000])
@pytest.mark.parametrize("page", [2, 8, 16, 32])
def test_prefill_block_shapes(qa, gpu, act, max_len, page):
    """rows and infinite values of every block shape on bf16 pages, a page missing"""
    p = Paged(67, [1, 70, 33, 190, 64, 150], new=[1, 70, 0, 131, 2, 97], group=2, kv_heads=2, page=page, act=act,
              cache="bf16", front=3, back=5)
    p.table[3, 64 // page] = p.n_pages
    p.v[p.page_of(5, 80), 1, 80 % page, 9] = math.inf
    p.v[p.page_of(5, 130), 1, 130 % page, 9] = math.nan
    check(p.gpu(qa).attention(qa, SCALE, max_len=max_len), *p.reference(SCALE))


@pytest.mark.parametrize("act,cache", TYPES)
def test_prefill_long_walk(qa, gpu, act, cache):
    """one block walks 9000 keys: the page ids are read more than once"""
    p = Paged(68, [9000], new=[3], group=2, kv_heads=1, page=16, act=act, cache=cache)
    p.table[0, 300] = -1
    check(p.gpu(qa).attention(qa, SCALE, max_len=64), *p.reference(SCALE))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("page", [2, 8, 16, 64])
def test_prefill_short_chunks(qa, gpu, act, cache, page):
    """a few rows each behind pasts, split and unsplit, with what the masks leave out undefined"""
    p = Paged(69, [500, 33, 129, 0, 64], new=[31, 2, 17, 0, 12], group=2, kv_heads=2, page=page, act=act, cache=cache, front=1)
    p.table[0, 96 // page] = -7
    p.v[p.page_of(2, 118), 1, 118 % page, 9] = -math.inf
    p.gpu(qa)
    for max_len in (64, 500, 3000):
        check(p.attention(qa, SCALE, max_len=max_len), *p.reference(SCALE))

"""Attention over a window and of trees of drafts, and rows that turn by given positions, through the C ABI on
device memory, against their definitions in 64 bits (tests/masks_util.py, which derives the tolerances)."""
import ctypes as C
import math

import pytest
import torch as T

import masks_util as M
import paged_util as U
from paged_util import HD, Paged, check

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(HD)
TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")]
LENS = [0, 1, 15, 16, 17, 63, 64, 65, 200, 530]


def check_window(qa, p, win, sinks, **k):
    check(M.window(qa, p, SCALE, win, sinks, **k), *M.reference(p, SCALE, M.window_sees(win, sinks), M.by_matrix(p)))


def spoil(p, sees, value=math.nan):
    """positions that no row sees hold `value`, as do their keys"""
    for s, (l, n) in enumerate(zip(p.lens, p.counts)):
        pos = T.arange(max(l, 0))
        seen = T.zeros(max(l, 0), dtype=T.bool)
        for i in range(n):
            seen |= sees(s, i, pos, max(l, 0) - n + i, max(l, 0) - n)
        for x in pos[~seen].tolist():
            at = p.page_of(s, x)
            if at >= 0:
                p.k[at, :, x % p.page] = value
                p.v[at, :, x % p.page] = value


# ---------------------------------------------------------------------------
# windows: single tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 9])
@pytest.mark.parametrize("win,sinks", [(1, 0), (64, 4), (100, 33)])
def test_window_tokens(qa, gpu, act, cache, group, win, sinks):
    """what is outside of the window and the first positions is no number"""
    p = Paged(110 + group, LENS, group=group, kv_heads=2, page=16, act=act, cache=cache)
    spoil(p, M.window_sees(win, sinks))
    check_window(qa, p.gpu(qa), win, sinks)


@pytest.mark.parametrize("win,sinks", [(1, 1), (2, 0), (31, 1), (32, 32), (33, 31), (512, 0), (1000, 4), (7, 600), (1, 529)])
@pytest.mark.parametrize("cache,group", [("f32", 2), ("bf16", 2), ("bf16", 8)])
def test_window_sizes(qa, gpu, win, sinks, cache, group):
    p = Paged(120, LENS, group=group, kv_heads=1, page=32, cache=cache)
    spoil(p, M.window_sees(win, sinks), math.inf)
    check_window(qa, p.gpu(qa), win, sinks)


@pytest.mark.parametrize("page", [1, 2, 8, 512])
@pytest.mark.parametrize("cache,group", [("f32", 2), ("bf16", 2), ("bf16", 6)])
def test_window_pages(qa, gpu, page, cache, group):
    """pages that no window reaches are given back"""
    win, sinks = 70, 5
    p = Paged(121, LENS, group=group, kv_heads=2, page=page, cache=cache)
    for s, l in enumerate(p.lens):
        for e in range(-(-l // page)):
            if (e + 1) * page <= l - win and e * page >= sinks:
                p.table[s, e] = -1
    check_window(qa, p.gpu(qa), win, sinks)


@pytest.mark.parametrize("max_len", [0, 1, 64, 300, 2 ** 31 - 1])
@pytest.mark.parametrize("packed", [False, True])
def test_window_any_max_len(qa, gpu, max_len, packed):
    p = Paged(122, [1, 900, 130, 0], new=[1, 3, 130, 0] if packed else None, group=2, kv_heads=2, page=32)
    check_window(qa, p.gpu(qa), 200, 10, max_len=max_len)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("packed", [False, True])
def test_window_of_everything(qa, gpu, act, cache, packed):
    """a window of all positions, or all of them as first ones, is attention without one: the same bits for
    single tokens; packed rows may be split otherwise, so both are within the tolerance of the definition"""
    new = [5, 100, 64, 2] if packed else None
    p = Paged(123, [300, 100, 64, 40], new=new, group=2, kv_heads=2, page=16, act=act, cache=cache).gpu(qa)
    want = p.attention(qa, SCALE)
    big = 2 ** 31 - 1
    tol = M.reference(p, SCALE, M.window_sees(big, 0), packed)[1]
    for win, sinks in ((big, 0), (big, big), (300, 0), (1, big)):
        got = M.window(qa, p, SCALE, win, sinks)
        if packed:
            assert bool(((got.double() - want.double()).abs().cpu() <= 2 * tol).all()), (win, sinks)
        else:
            assert T.equal(got, want), (win, sinks)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_window_missing_pages(qa, gpu, packed, cache):
    """pages that are none inside the window, among the first positions and everywhere"""
    p = Paged(124, [300, 100, 64, 40], new=[5, 100, 64, 2] if packed else None, group=2, kv_heads=2, page=16, cache=cache)
    p.table[0, 0] = -1
    p.table[0, 16] = p.n_pages
    p.table[1, 3] = 2 ** 31 - 1
    p.table[2, :] = -2 ** 31
    check_window(qa, p.gpu(qa), 90, 20)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("cache,group", [("f32", 2), ("bf16", 5)])
def test_window_longer_than_the_table(qa, gpu, packed, cache, group):
    """a length past the page table's end: the window's positions in the table and the first ones are seen"""
    p = Paged(125, [100, 60, 50], new=[30, 8, 3] if packed else None, group=group, kv_heads=1, page=8, cache=cache)
    p.table = p.table[:, :6].contiguous()          # 48 positions
    check_window(qa, p.gpu(qa), 20, 3)
    for l in (2 ** 31 - 1, 2 ** 30 + 7):
        p.lens[0] = l
        p.kv_len[0] = l
        p.d["kv_len"].copy_(p.kv_len)
        check_window(qa, p, 20, 3)
        check_window(qa, p, 2 ** 31 - 1, 0)


# ---------------------------------------------------------------------------
# windows: packed rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("group,kv_heads", [(1, 2), (2, 2), (3, 1), (8, 1)])
@pytest.mark.parametrize("win,sinks", [(1, 0), (40, 7), (97, 64)])
def test_window_packed(qa, gpu, act, cache, group, kv_heads, win, sinks):
    """prompts from one row to several tiles behind pasts, a sequence without rows between and rows of no
    sequence around; what no row sees is no number"""
    p = Paged(140 + group, [1, 70, 33, 190, 64, 250], new=[1, 70, 0, 131, 2, 97], group=group, kv_heads=kv_heads, page=16,
              act=act, cache=cache, front=3, back=5)
    spoil(p, M.window_sees(win, sinks))
    check_window(qa, p.gpu(qa), win, sinks)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 256])
def test_window_packed_pages(qa, gpu, act, cache, page):
    """every page size's path, with what earlier rows of the window see infinite or none"""
    p = Paged(150, [31, 390, 33, 205], new=[31, 290, 33, 5], group=2, kv_heads=2, page=page, act=act, cache=cache)
    p.v[p.page_of(1, 150), 1, 150 % page, 9] = math.inf
    p.v[p.page_of(1, 200), 0, 200 % page, 3] = math.nan
    p.k[p.page_of(1, 300), 0, 300 % page, 3] = math.nan
    check_window(qa, p.gpu(qa), 75, 3)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("max_len", [64, 700, 5000])
def test_window_packed_split(qa, gpu, act, cache, max_len):
    """both block shapes, with and without a split over the keys"""
    p = Paged(151, [1024, 700, 65, 1300], new=[31, 2, 65, 150], group=2, kv_heads=2, page=16, act=act, cache=cache, back=2)
    for win, sinks in ((600, 40), (33, 0), (2000, 0)):
        check_window(qa, p.gpu(qa), win, sinks, max_len=max_len)


def test_window_packed_more_rows_than_positions(qa, gpu):
    p = Paged(152, [3, 0, -4, 40], new=[5, 4, 2, 40], group=2, kv_heads=2, page=8, back=1).gpu(qa)
    check_window(qa, p, 2, 1)


def test_window_many_sequences(qa, gpu):
    lens = [(5 * i) % 61 + 1 for i in range(200)]
    p = Paged(153, lens, new=[min(l, i % 3) for i, l in enumerate(lens)], group=2, kv_heads=1, page=4, front=2).gpu(qa)
    check_window(qa, p, 9, 2)


def test_window_long_walk(qa, gpu):
    """one block walks more tiles than page ids are read at a time, the gap inside"""
    p = Paged(154, [9000], new=[3], group=2, kv_heads=1, page=16, cache="bf16")
    check_window(qa, p.gpu(qa), 5000, 2500, max_len=64)


# ---------------------------------------------------------------------------
# trees
# ---------------------------------------------------------------------------
def check_tree(qa, p, bits, words, **k):
    seen = [[b & ((1 << 64 * words) - 1) for b in s] for s in bits]
    check(M.tree(qa, p, SCALE, bits, words, **k), *M.reference(p, SCALE, M.tree_sees(seen), True))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("group,kv_heads", [(1, 2), (2, 2), (3, 1), (8, 1), (16, 1)])
def test_tree(qa, gpu, act, cache, group, kv_heads):
    """trees of one draft to 64 behind pasts of none to several tiles; drafts that no row sees are no number"""
    new = [1, 17, 0, 64, 33, 6]
    p = Paged(160 + group, [1, 70, 33, 164, 33, 250], new=new, group=group, kv_heads=kv_heads, page=16, act=act, cache=cache,
              front=3, back=5)
    bits = [M.random_tree(p.g, n) for n in new]
    bits[3] = [b & ~(1 << 40) for b in bits[3]]
    spoil(p, M.tree_sees(bits))
    check_tree(qa, p.gpu(qa), bits, 1)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("words,n", [(1, 64), (2, 65), (2, 128), (3, 130), (4, 256)])
def test_tree_words(qa, gpu, act, cache, words, n):
    """any bits, in every word; the past ends inside a tile"""
    p = Paged(170, [n + 45, n], new=[n, n], group=2, kv_heads=1, page=16, act=act, cache=cache)
    bits = [[int(T.randint(0, 2 ** 62, (1,), generator=p.g)) * 5 ** (i % 90) & ((1 << n) - 1) for i in range(n)] for _ in range(2)]
    check_tree(qa, p.gpu(qa), bits, words)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("bf16", "bf16")])
def test_tree_empty_rows(qa, gpu, act, cache):
    """rows without bits: the past alone; with no past: 0.  Bits of drafts that are not there mean nothing"""
    p = Paged(171, [20, 5, 40], new=[20, 5, 7], group=2, kv_heads=2, page=8, act=act, cache=cache)
    bits = [[0 if i % 3 else 1 << i for i in range(20)], [0] * 5, [(2 ** 64 - 1) ^ (1 << i) for i in range(7)]]
    check_tree(qa, p.gpu(qa), bits, 1)


def test_tree_more_drafts_than_bits(qa, gpu):
    """drafts behind the last bit are seen by no row"""
    p = Paged(172, [300], new=[150], group=2, kv_heads=1, page=16, cache="bf16")
    bits = [[(1 << i + 1) - 1 for i in range(150)]]
    check_tree(qa, p.gpu(qa), bits, 1)
    check_tree(qa, p, bits, 2)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 128])
@pytest.mark.parametrize("act,cache", TYPES)
def test_tree_pages(qa, gpu, act, cache, page):
    new = [31, 3, 33, 5]
    p = Paged(173, [31, 190, 133, 205], new=new, group=2, kv_heads=2, page=page, act=act, cache=cache)
    p.table[1, 100 // page] = -1
    p.table[3, 203 // page] = p.n_pages
    p.v[p.page_of(2, 110), 1, 110 % page, 9] = math.inf      # a draft that some rows see
    check_tree(qa, p.gpu(qa), [M.random_tree(p.g, n) for n in new], 1)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("max_len", [0, 64, 700, 5000])
def test_tree_split(qa, gpu, act, cache, max_len):
    new = [31, 2, 64, 150]
    p = Paged(174, [1024, 700, 65, 1300], new=new, group=2, kv_heads=2, page=16, act=act, cache=cache, back=2)
    check_tree(qa, p.gpu(qa), [M.random_tree(p.g, n) for n in new], 3, max_len=max_len)


def test_tree_more_rows_than_positions(qa, gpu):
    """drafts at negative positions are not there; the others are seen by their bits"""
    new = [5, 4, 2, 40]
    p = Paged(175, [3, 0, -4, 40], new=new, group=2, kv_heads=2, page=8, back=1).gpu(qa)
    check_tree(qa, p, [[(1 << n) - 1] * n for n in new], 1)


def test_tree_of_one_draft_each(qa, gpu):
    """without row_start: one draft a sequence"""
    p = Paged(176, LENS, group=2, kv_heads=2, page=16, cache="bf16").gpu(qa)
    check_tree(qa, p, [[1] for _ in LENS], 1)


def test_tree_many_sequences(qa, gpu):
    lens = [(5 * i) % 61 + 7 for i in range(200)]
    new = [i % 7 for i in range(200)]
    p = Paged(177, lens, new=new, group=2, kv_heads=1, page=4, front=2).gpu(qa)
    check_tree(qa, p, [M.random_tree(p.g, n, 3) for n in new], 2)


def test_tree_of_one_branch_is_a_prompt(qa, gpu):
    """a chain's bits are the causal mask: within both tolerances"""
    new = [64, 30]
    p = Paged(178, [500, 30], new=new, group=2, kv_heads=2, page=16, cache="bf16").gpu(qa)
    bits = [[(1 << i + 1) - 1 for i in range(n)] for n in new]
    x, y = M.tree(qa, p, SCALE, bits, 1).double(), p.attention(qa, SCALE).double()
    tol = M.reference(p, SCALE, M.tree_sees(bits), True)[1]
    assert bool(((x - y).abs().cpu() <= 2 * tol).all())


# ---------------------------------------------------------------------------
# rows that turn by given positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act,cache", TYPES)
def test_append_at(qa, gpu, act, cache):
    """rows sit one behind the other and turn by their own positions; rows at negative or missing places, or with
    positions outside the tables, are left out"""
    new = [5, 7, 0, 9, 4]
    p = Paged(180, [5, 40, 16, 33, 3], new=new, group=3, kv_heads=2, page=8, act=act, cache=cache, front=2, back=3)
    p.table[3, 3] = -1
    g, H, KH, n_pos = p.g, p.heads, p.kv_heads, 50
    dt = U.T[act]
    turn = T.randint(0, n_pos, (p.rows,), generator=g).to(T.int32)
    turn[p.starts[1] + 2], turn[p.starts[1] + 3], turn[p.starts[3]] = -1, n_pos, 2 ** 31 - 1
    q, k, v = T.randn(p.rows, H * HD, generator=g).to(dt), *(T.randn(p.rows, KH * HD, generator=g).to(dt) for _ in range(2))
    wq, wk = (1 + 0.1 * T.randn(HD, generator=g) for _ in range(2))
    cos, sin = U.rope_tables(n_pos)
    p.gpu(qa)
    d = [x.cuda() for x in (turn, q, k, v, wq, wk, cos, sin)]
    out = T.full_like(d[1], 7.0)
    qa.check(qa.lib().qwen_hip_paged_append_at(
        C.byref(p.c_kv), C.byref(p.c_batch), d[0].data_ptr(), out.data_ptr(), d[1].data_ptr(), d[2].data_ptr(),
        d[3].data_ptr(), p.c_act, H * HD, KH * HD, H, d[4].data_ptr(), d[5].data_ptr(), 1e-6, d[6].data_ptr(),
        d[7].data_ptr(), n_pos, None), "append_at")
    T.cuda.synchronize()
    want_q, want_k, want_v = T.full((p.rows, H, HD), 7.0, dtype=T.float64), p.k.double(), p.v.double()
    tol_q, tol_k, e = T.zeros_like(want_q), T.zeros_like(want_k), 20 * 2.0 ** -24      # test_gpu_paged.run_append derives it
    for s, (l, n) in enumerate(zip(p.lens, new)):
        for i in range(n):
            row, pos = p.starts[s] + i, l - n + i
            by = int(turn[row])
            if pos < 0 or not 0 <= by < n_pos:
                continue
            for x, w, heads in ((q, wq, H), (k, wk, KH)):
                y = U.norm_rope(x[row].view(heads, HD), w, 1e-6, cos[by], sin[by])
                size = T.maximum(*(U.norm_rope(x[row].view(heads, HD).abs(), w.abs(), 1e-6, cos[by].abs(), f * sin[by].abs())
                                   for f in (-1, 1)))
                pid = p.page_of(s, pos)
                if heads == H and x is q:
                    want_q[row], tol_q[row] = y, e * size + U.HALF[act] * y.abs()
                elif pid >= 0:
                    want_k[pid, :, pos % 8], tol_k[pid, :, pos % 8] = y, e * size + U.HALF[cache] * y.abs()
                    want_v[pid, :, pos % 8] = v[row].view(KH, HD).to(U.T[cache]).double()
    for got, want, tol in ((out.cpu().view(p.rows, H, HD), want_q, tol_q), (p.d["k"].cpu(), want_k, tol_k),
                           (p.d["v"].cpu(), want_v, T.zeros_like(want_v))):
        got = got.double()
        assert bool((((got - want).abs() <= tol) | (T.isnan(got) & T.isnan(want))).all())


# ---------------------------------------------------------------------------
# streams
# ---------------------------------------------------------------------------
def test_two_streams(qa, gpu):
    """two calls that may overlap, a workspace each"""
    new = [31, 2, 40]
    a = Paged(190, [1024, 700, 500], group=2, kv_heads=2, page=16).gpu(qa)
    b = Paged(191, [1024, 700, 500], new=new, group=2, kv_heads=2, page=16, act="bf16", cache="bf16").gpu(qa)
    bits = [M.random_tree(b.g, n) for n in new]
    L, st = qa.lib(), [T.cuda.Stream() for _ in range(2)]
    ab, bb = ((C.byref(x.c_kv), C.byref(x.c_batch)) for x in (a, b))
    na, nb = L.qwen_hip_paged_attention_window_ws_bytes(*ab, 4, 400, 30), L.qwen_hip_paged_attention_tree_ws_bytes(*bb, 4)
    wa, wb = (T.empty(max(n, 16), dtype=T.uint8, device="cuda") for n in (na, nb))
    tree = M.tree_words(b, bits, 1).cuda()
    oa, ob = (T.full_like(x.d["q"], 7.0) for x in (a, b))
    T.cuda.synchronize()
    for _ in range(5):
        qa.check(L.qwen_hip_paged_attention_window(*ab, oa.data_ptr(), a.d["q"].data_ptr(), a.c_act, 4, SCALE, 400, 30,
                                                   wa.data_ptr(), na, st[0].cuda_stream))
        qa.check(L.qwen_hip_paged_attention_tree(*bb, ob.data_ptr(), b.d["q"].data_ptr(), b.c_act, 4, SCALE, tree.data_ptr(), 1,
                                                 wb.data_ptr(), nb, st[1].cuda_stream))
    T.cuda.synchronize()
    check(oa, *M.reference(a, SCALE, M.window_sees(400, 30), False))
    check(ob, *M.reference(b, SCALE, M.tree_sees(bits), True))

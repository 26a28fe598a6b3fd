"""Page tables that continue others, copies of pages and accepted drafts in several layers, through the C ABI on
device memory, against their definitions (tests/pages_util.py): whole numbers and bits, all exact."""
import ctypes as C
import random

import pytest
import torch as T

import pages_util as G
from pages_util import HD

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# fork
# ---------------------------------------------------------------------------
def same_fork(qa, table, lens, parent, new, outside, page, n_pages):
    n = len(parent) if parent is not None else len(table)
    want = G.fork_reference(table, lens, list(range(n)) if parent is None else parent, [0] * n if new is None else new,
                            outside, page, n_pages)
    got = G.fork(qa, table, lens, parent, new, outside, page, n_pages)
    for what, a, b in zip(("table", "lengths", "copies", "missing"), got, want):
        assert a == b, what
    return got


def beams(rng, seqs, n, page, longest, apart, stride, n_pages):
    """a table of beams that share their first pages, in any order of ids"""
    ids = list(range(n_pages))
    rng.shuffle(ids)
    table, lens = [], []
    for _ in range(seqs):
        l = rng.randint(1, longest)
        common = [ids.pop() for _ in range(max(0, l - apart) // page)]
        for _ in range(n):
            own = [ids.pop() for _ in range(-(-l // page) - len(common))]
            table.append((common + own + [-1] * stride)[:stride])
            lens.append(l)
    return table, lens


@pytest.mark.parametrize("page", [1, 2, 16, 64])
@pytest.mark.parametrize("seed", range(4))
def test_fork_beams(qa, gpu, page, seed):
    """beams continue chosen beams, some with several continuations, some with none; new rows of none to several pages"""
    rng = random.Random(seed)
    stride = 200 // page + 4
    table, lens = beams(rng, 5, 4, page, 190, 30, stride, 1700)
    parent = [4 * (i // 4) + rng.randrange(4) for i in range(20)]
    parent[rng.randrange(20)] = -1
    parent[rng.randrange(20)] = rng.choice([20, 2 ** 31 - 1, -2 ** 31])
    new = [rng.choice([1, 1, 1, 0, 3, 2 * page + 1, -5]) for _ in range(20)]
    same_fork(qa, table, lens, parent, new, [], page, 1700)


@pytest.mark.parametrize("held", [[], [0, 31, 32, 40], list(range(0, 96, 2))])
def test_fork_rules(qa, gpu, held):
    """who keeps a page: the row with the most positions in it, of several the last; none where a row has it for positions
    behind or the program holds it; a row without new rows leaves its own"""
    a, b, c = 40, 41, 42
    table = [[a, b, -1, -1], [a, b, c, -1], [a, -1, -1, -1], [-1, b, -1, -1], [a, 96, 7, -1], [-1] * 4, [a, -1, -1, -1]]
    lens = [24, 40, 10, 20, 32, 0, 12]
    n = len(lens)
    for parent in ([2, 6], [6, 2], [6, 2, 2], [2, 6, 6, 2], [0, 0, 0], [0, 1, 0], [2, 2, 2, 0], [2, 2], [3, 3, 3], [1, 1, 0, 0, 2, 2, 3, 5, -1], [4, 4, 4], list(range(n)), None):
        rows = n if parent is None else len(parent)
        for new in (None, [1] * rows, [0] * (rows - 1) + [5], [(9 * i) % 20 for i in range(rows)], [16] * rows):
            same_fork(qa, table, lens, parent, new, held, 16, 96)


def test_fork_missing(qa, gpu):
    """fewer free pages than rows want: the first rows get them, a copy that has no page is no copy; rows longer than the
    table"""
    table = [[0, 1, -1, -1], [2, 3, -1, -1], [4, -1, -1, -1]]
    for n_pages in (5, 6, 7, 8, 12):
        for lens in ([8, 7, 3], [6, 5, 4], [30, 16, 4], [2 ** 31 - 1, 15, 0]):
            for parent in ([0, 0, 1, 1, 2], [1, 1, 1, 1], [2, 0, -1]):
                for k in (1, 9, 2 ** 31 - 1):
                    same_fork(qa, table, lens, parent, [k] * len(parent), [], 4, n_pages)


def test_fork_bad_ids(qa, gpu):
    """ids outside the pages are none: they come out as -1, and a last page that is none is taken fresh"""
    table = [[5, -7, 2 ** 31 - 1, 9], [10, 3, 12, -2 ** 31]]
    for lens in ([13, 15], [12, 16], [-3, 6]):
        for parent in ([0, 1, 0, 1], [1, 1, 0]):
            same_fork(qa, table, lens, parent, [2] * len(parent), [], 4, 10)


@pytest.mark.parametrize("n_pages", [1, 31, 32, 33, 1 << 16, (1 << 16) + 1, 1 << 19, (1 << 19) + 1, (1 << 20) + 5])
def test_fork_page_counts(qa, gpu, n_pages):
    """bits in LDS of both sizes and in the workspace; the last pages among them"""
    rng = random.Random(n_pages)
    used = sorted({0, n_pages - 1, n_pages // 2, min(40, n_pages - 1)})
    table = [(used[:2] + [-1] * 8)[:8], (used[2:] + [-1] * 8)[:8]]
    lens = [2 * 4 - 1 if len(used) > 1 else 3, 4 * len(used[2:])]
    same_fork(qa, table, lens, [0, 0, 1, -1, 1], [1, 5, 9, 20, 1], [], 4, n_pages)
    if n_pages > 1000:
        # nearly all pages held: the free ones lie far apart
        free = set(rng.sample(range(n_pages), 9))
        same_fork(qa, table, lens, [0, 0, 1, -1, 1], [1, 5, 9, 20, 1], [i for i in range(n_pages) if i not in free], 4, n_pages)


def test_fork_many_rows(qa, gpu):
    """the most rows of a call, long tables"""
    rng = random.Random(9)
    table, lens = beams(rng, 128, 8, 8, 600, 20, 90, 20000)
    parent = [8 * (i // 8) + min(rng.randrange(8), rng.randrange(8)) for i in range(1024)]
    same_fork(qa, table, lens, parent, [1] * 1024, [], 8, 20000)
    same_fork(qa, table[:3], lens[:3], [0] * 1024, [2] * 1024, [], 8, 20000)


def test_fork_from_no_table(qa, gpu):
    """the first sequences: pages for their prompts"""
    n = 3
    kv = qa.PagedKV(None, None, None, qa.ST_F32, 20, 4, 2, HD, 0, 5)
    new = T.tensor([9, 0, 4], dtype=T.int32, device="cuda")
    parent = T.full((n,), -1, dtype=T.int32, device="cuda")
    out, ln, cp, ms = (T.full(s, 7, dtype=T.int32, device="cuda") for s in ((n, 5), (n,), (n, 4), (1,)))
    qa.check(qa.lib().qwen_hip_paged_fork(C.byref(kv), None, parent.data_ptr(), new.data_ptr(), None, n, out.data_ptr(),
                                          ln.data_ptr(), cp.data_ptr(), ms.data_ptr(), None, 0, None))
    T.cuda.synchronize()
    assert out.tolist() == [[0, 1, 2, -1, -1], [-1] * 5, [3, -1, -1, -1, -1]] and ln.tolist() == [9, 0, 4]
    assert cp.tolist() == [[-1, -1, 0, 0]] * n and int(ms) == 0


@pytest.mark.parametrize("waiting", [False, True])
def test_fork_step_by_step(qa, gpu, waiting):
    """beams over many steps: what a row's positions hold is what its ancestors wrote; `waiting`: some rows stand still for
    steps (no new rows) while others of the same past go on, in any order"""
    rng, page, n_pages, stride = random.Random(5), 4, 120, 16
    for start in range(8 if waiting else 1):
        table, lens = [[-1] * stride], [0]
        table, lens, _, miss = G.fork(qa, table, lens, [0], [6], [], page, n_pages)
        assert miss == 0
        store = {}                                         # (page, slot) -> what a row wrote
        said = [[("prompt", i) for i in range(6)]]
        for i in range(6):
            store[table[0][i // page], i % page] = said[0][i]
        for step in range(40):
            n = rng.choice([1, 3, 6]) if not waiting else rng.choice([3, 6, 8])
            parent = [rng.randrange(len(table)) for _ in range(n)]
            new = [rng.choice([0, 0, 1, 2]) if waiting else 1 for _ in range(n)]
            table, lens, copies, miss = same_fork(qa, table, lens, parent, new, [], page, n_pages)
            assert miss == 0
            for a, b, first, slots in copies:
                for i in range(first, first + slots):
                    store[b, i] = store[a, i]
            said = [said[p] + [(step, s, i) for i in range(new[s])] for s, p in enumerate(parent)]
            for s in range(n):
                for i in range(lens[s] - new[s], lens[s]):
                    store[table[s][i // page], i % page] = said[s][i]
            for s in range(n):
                assert [store[table[s][i // page], i % page] for i in range(lens[s])] == said[s], (start, step, s)
            if max(lens) > 50:
                break


# ---------------------------------------------------------------------------
# copies and accepted drafts
# ---------------------------------------------------------------------------
class Layers:
    def __init__(self, qa, L, n_pages, kv_heads, page, cache, table=None, seed=0):
        g = T.Generator().manual_seed(seed)
        self.pages = T.randn(L, 2, n_pages, kv_heads, page, HD, generator=g).to(G.T[cache])
        self.d = self.pages.cuda()
        self.table = T.tensor(table if table is not None else [[0]], dtype=T.int32, device="cuda")
        code = {"f32": qa.ST_F32, "bf16": qa.ST_BF16}[cache]
        self.c = (qa.PagedKV * L)(*[qa.PagedKV(p[0].data_ptr(), p[1].data_ptr(), self.table.data_ptr(), code, n_pages, page,
                                               kv_heads, HD, *self.table.shape) for p in self.d])
        self.L = L


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("L,kv_heads,page", [(1, 1, 1), (3, 2, 16), (28, 8, 4), (64, 1, 8), (2, 5, 256)])
def test_copy(qa, gpu, cache, L, kv_heads, page):
    n_pages = 9
    x = Layers(qa, L, n_pages, kv_heads, page, cache)
    copies = [[0, 1, 0, page], [0, 2, page - 1, 1], [3, 4, 0, max(page // 2, 1)], [3, 3, 0, page], [-1, 5, 0, page], [6, n_pages, 0, 1],
              [6, -1, 0, 1], [n_pages, 5, 0, 1], [6, 5, 0, 0], [6, 5, -1, 1], [6, 5, 0, page + 1], [6, 5, 1, page],
              [6, 5, 0, 2 ** 31 - 1], [6, 5, 2 ** 31 - 1, 1], [7, 8, page // 2, page - page // 2]]
    want = x.pages.clone()
    for a, b, f, n in copies:
        if 0 <= a < n_pages and 0 <= b < n_pages and f >= 0 and n > 0 and f + n <= page:
            want[:, :, b, :, f:f + n] = x.pages[:, :, a, :, f:f + n]
    c = T.tensor(copies, dtype=T.int32, device="cuda")
    qa.check(qa.lib().qwen_hip_paged_copy(x.c, L, c.data_ptr(), len(copies), None))
    T.cuda.synchronize()
    assert T.equal(x.d.cpu(), want)


def compact_reference(x, table, starts, lens, path, count, page):
    n_pages, stride = x.shape[2], len(table[0])
    done, out = x.clone(), []
    def place(s, p):
        if not 0 <= p < stride * page or not 0 <= table[s][p // page] < n_pages:
            return None
        return table[s][p // page], p % page
    for s in range(len(lens)):
        n = starts[s + 1] - starts[s]
        past, got = max(lens[s], 0) - n, 0
        for i in range(max(0, min(count[s], len(path[s]), n))):
            d = path[s][i]
            if d >= n or d <= (path[s][i - 1] if i else -1):
                break
            a, b = place(s, past + d), place(s, past + i)
            if a and b:
                done[:, :, b[0], :, b[1]] = x[:, :, a[0], :, a[1]]
            got += 1
        out.append(max(past + got, 0))
    return done, out


def same_compact(qa, x, table, starts, lens, path, count, page, row_start=True, max_len=0):
    ints = lambda v: T.tensor(v, dtype=T.int32, device="cuda")
    d = [ints(v) for v in (starts, lens, path, count)]
    out = T.full((len(lens),), 7, dtype=T.int32, device="cuda")
    b = qa.PagedBatch(d[0].data_ptr() if row_start else None, d[1].data_ptr(), starts[-1] if row_start else len(lens), max_len)
    want, want_len = compact_reference(x.d.cpu(), table, starts, lens, path, count, page)
    T.cuda.synchronize()
    qa.check(qa.lib().qwen_hip_paged_compact(x.c, x.L, C.byref(b), out.data_ptr(), d[2].data_ptr(), len(path[0]),
                                             d[3].data_ptr(), None))
    T.cuda.synchronize()
    assert out.tolist() == want_len
    assert T.equal(x.d.cpu(), want)


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("L,kv_heads,page", [(1, 1, 1), (3, 2, 16), (28, 8, 4), (64, 1, 8), (2, 20, 32)])
def test_compact(qa, gpu, cache, L, kv_heads, page):
    """paths of all kinds: none, all, chains, gaps; over page borders; sequences without drafts"""
    rng = random.Random(page)
    news, lens = [16, 1, 0, 64, 33, 5], [50, 1, 20, 64, 70, 9]
    n_pages = sum(-(-l // page) for l in lens) + 2
    ids = list(range(n_pages))
    rng.shuffle(ids)
    stride = -(-70 // page)
    table = [([ids.pop() for _ in range(-(-l // page))] + [-1] * stride)[:stride] for l in lens]
    path, count = [], []
    for n in news:
        k = rng.randint(0, n)
        path.append((sorted(rng.sample(range(n), k)) + [0] * 64)[:64])
        count.append(k)
    path[3], count[3] = list(range(64)), 64
    starts = [2]
    for n in news:
        starts.append(starts[-1] + n)
    x = Layers(qa, L, n_pages, kv_heads, page, cache, table)
    same_compact(qa, x, table, starts, lens, path, count, page)


def test_compact_long_paths(qa, gpu):
    """more accepted drafts than a block takes at a time"""
    rng = random.Random(3)
    table = [[i for i in range(100)]]
    x = Layers(qa, 2, 100, 2, 16, "bf16", table)
    path = sorted(rng.sample(range(1200), 700))
    same_compact(qa, x, table, [0, 1200], [1500], [path], [700], 16)


def test_compact_bad_paths(qa, gpu):
    """lists end at what is no draft or not above the one before; counts past the list or below zero; pages that are none;
    drafts at negative positions; a table that is too short"""
    table = [[0, 1, 2, -1], [3, 4, 5, 6], [7, 99, 8, -1], [9, 10, -1, -1], [11, 12, 13, 14]]
    lens, starts = [12, 16, 12, 2, 30], [0, 6, 14, 22, 27, 39]
    for path in ([1, 3, 3, 4, 5], [2, 1, 4, 5, 5], [0, 1, 6, 7, 8], [-1, 2, 3, 4, 5], [1, 2, 3, 4, 2 ** 31 - 1], [2 ** 31 - 1] * 5, [3, 4, 5, 6, 7]):
        for count in (5, 3, 2 ** 31 - 1, -1, 0):
            x = Layers(qa, 2, 15, 2, 4, "f32", table)
            same_compact(qa, x, table, starts, lens, [path] * 5, [count] * 5, 4)


def test_compact_single_rows(qa, gpu):
    """without row_start a sequence has one draft: taken or not"""
    table = [[0, 1], [2, 3], [4, 5]]
    x = Layers(qa, 1, 6, 1, 4, "f32", table)
    same_compact(qa, x, table, [0, 1, 2, 3], [5, 8, 0], [[0], [0], [0]], [1, 0, 1], 4, row_start=False)


def test_two_streams(qa, gpu):
    """fork and copy on one stream beside accepted drafts of other caches on another"""
    st = [T.cuda.Stream() for _ in range(2)]
    table = [[0, 1, 2], [3, 4, 5]]
    x, y = Layers(qa, 8, 12, 2, 16, "bf16", table), Layers(qa, 8, 6, 2, 16, "f32", table, seed=1)
    ints = lambda v: T.tensor(v, dtype=T.int32, device="cuda")
    lens, parent, new = ints([40, 39]), ints([0, 0, 1, 0]), ints([1] * 4)
    out, ln, cp, ms = (T.zeros(s, dtype=T.int32, device="cuda") for s in ((4, 3), (4,), (4, 4), (1,)))
    starts, path, count, ln2 = ints([0, 9, 18]), ints([[1, 4, 7], [0, 2, 8]]), ints([3, 2]), ints([0, 0])
    b = qa.PagedBatch(starts.data_ptr(), lens.data_ptr(), 18, 0)
    want = compact_reference(y.pages, table, [0, 9, 18], [40, 39], path.tolist(), [3, 2], 16)
    ref = G.fork_reference(table, [40, 39], [0, 0, 1, 0], [1] * 4, [], 16, 12)
    T.cuda.synchronize()
    L = qa.lib()
    qa.check(L.qwen_hip_paged_fork(x.c, lens.data_ptr(), parent.data_ptr(), new.data_ptr(), None, 4, out.data_ptr(), ln.data_ptr(),
                                   cp.data_ptr(), ms.data_ptr(), None, 0, st[0].cuda_stream))
    qa.check(L.qwen_hip_paged_compact(y.c, 8, C.byref(b), ln2.data_ptr(), path.data_ptr(), 3, count.data_ptr(), st[1].cuda_stream))
    qa.check(L.qwen_hip_paged_copy(x.c, 8, cp.data_ptr(), 4, st[0].cuda_stream))
    T.cuda.synchronize()
    assert (out.tolist(), ln.tolist(), cp.tolist(), int(ms)) == ref
    done = x.pages.clone()
    for a, to, f, n in ref[2]:
        if a >= 0:
            done[:, :, to, :, f:f + n] = x.pages[:, :, a, :, f:f + n]
    assert T.equal(x.d.cpu(), done)
    assert ln2.tolist() == want[1] and T.equal(y.d.cpu(), want[0])

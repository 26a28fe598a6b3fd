"""The operators of streams with several continuations and of streams that do not end, together, as a program uses
them: beam search (selection, page tables that continue others, copies, append, attention), drafts of a tree that
are checked in one pass and accepted, and a stream that keeps a window's pages.  Each step is checked against the
definitions on the values that the run gave it, and what the cache holds against every continuation's own past."""
import ctypes as C
import math

import numpy as np
import pytest
import torch as T

import masks_util as M
import pages_util as G
import paged_util as U
from paged_util import HD

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(HD)
EPS = 1e-6
H, KH, HIDDEN, VOCAB, PAGE = 4, 2, 256, 1000, 8


class Model:
    """`L` layers of attention over one cache each, sharing one page table (no products between them but a
    projection): hidden rows -> Q|K|V -> append -> attention -> next layer; logits from the last"""

    def __init__(self, qa, cache, n_pages, stride, L=3):
        g = T.Generator().manual_seed(21)
        self.qa, self.L, self.cache, self.n_pages, self.stride = qa, L, cache, n_pages, stride
        w = lambda *s, std=0.06: (T.randn(*s, generator=g) * std).bfloat16().cuda()
        self.w_qkv = [w((H + 2 * KH) * HD, HIDDEN) for _ in range(L)]
        self.w_o = [w(HIDDEN, H * HD, std=0.2) for _ in range(L)]
        self.emb, self.head = w(VOCAB, HIDDEN, std=1.0), w(VOCAB, HIDDEN, std=0.3)
        self.qn, self.kn = ((1 + 0.1 * T.randn(HD, generator=g)).cuda() for _ in range(2))
        self.cos, self.sin = (x.cuda() for x in U.rope_tables(stride * PAGE))
        self.pages = T.full((L, 2, n_pages, KH, PAGE, HD), math.nan, dtype=U.T[cache], device="cuda")
        self.ws = T.empty(8 << 20, dtype=T.uint8, device="cuda")
        self.code = {"f32": qa.ST_F32, "bf16": qa.ST_BF16}[cache]

    def kv(self, table):
        return (self.qa.PagedKV * self.L)(*[self.qa.PagedKV(p[0].data_ptr(), p[1].data_ptr(), table.data_ptr(), self.code,
                                                            self.n_pages, PAGE, KH, HD, *table.shape) for p in self.pages])

    def linear(self, x, w):
        y = T.empty(x.shape[0], w.shape[0], device="cuda")
        self.qa.check(self.qa.lib().qwen_hip_linear_nobias_bf16_noalloc(
            y.data_ptr(), x.data_ptr(), w.data_ptr(), x.shape[0], x.shape[1], w.shape[0],
            T.cuda.current_stream().cuda_stream), "linear")
        return y

    def rows(self, tokens, table, lens, start=None, turn=None, tree=None, window=None):
        """logits of all rows; start: packed rows; turn, tree: drafts; window: (positions, first ones)"""
        qa, L, st = self.qa, self.qa.lib(), T.cuda.current_stream().cuda_stream
        kvs = self.kv(table)
        x = self.emb[tokens.long()].float().contiguous()
        n = x.shape[0]
        b = qa.PagedBatch(None if start is None else start.data_ptr(), lens.data_ptr(), n, 0)
        width = (H + 2 * KH) * HD
        self.seen = []
        for l in range(self.L):
            by = C.byref(kvs[l]), C.byref(b)
            qkv = self.linear(x, self.w_qkv[l])
            q, at = T.empty(n, H * HD, device="cuda"), qkv.data_ptr()
            rest = (q.data_ptr(), at, at + 4 * H * HD, at + 4 * (H + KH) * HD, qa.ST_F32, width, width, H, self.qn.data_ptr(),
                    self.kn.data_ptr(), EPS, self.cos.data_ptr(), self.sin.data_ptr(), self.cos.shape[0], st)
            if turn is None:
                qa.check(L.qwen_hip_paged_append(*by, *rest))
            else:
                qa.check(L.qwen_hip_paged_append_at(*by, turn.data_ptr(), *rest))
            out = T.empty_like(q)
            end = (self.ws.data_ptr(), self.ws.numel(), st)
            if tree is not None:
                qa.check(L.qwen_hip_paged_attention_tree(*by, out.data_ptr(), q.data_ptr(), qa.ST_F32, H, SCALE, tree.data_ptr(),
                                                         tree.shape[1], *end))
            elif window is not None:
                qa.check(L.qwen_hip_paged_attention_window(*by, out.data_ptr(), q.data_ptr(), qa.ST_F32, H, SCALE, *window, *end))
            else:
                call = L.qwen_hip_paged_attention_decode if start is None else L.qwen_hip_paged_attention_prefill
                qa.check(call(*by, out.data_ptr(), q.data_ptr(), qa.ST_F32, H, SCALE, *end))
            self.seen.append((q, out))
            x = self.linear(out, self.w_o[l])
        return self.linear(x, self.head)

    def check_attention(self, table, lens, new, sees, layer):
        """attention of a layer against its definition, from the pages and queries as the device has them"""
        p = U.Paged.__new__(U.Paged)
        p.lens, p.counts, p.group, p.kv_heads, p.heads, p.page = lens, new, H // KH, KH, H, PAGE
        p.act, p.cache, p.table, p.n_pages, p.rows = "f32", self.cache, table.cpu(), self.n_pages, sum(new)
        p.k, p.v, p.q, p.row_start = self.pages[layer, 0].cpu(), self.pages[layer, 1].cpu(), self.seen[layer][0].cpu(), None
        p.starts = [sum(new[:i]) for i in range(len(new) + 1)]
        U.check(self.seen[layer][1], *M.reference(p, SCALE, sees, True))

    def cached(self, table, s, n):
        """[layers][2][n][KH][HD]: what row s of the table holds of its first n positions"""
        t = table.cpu()[s].long()
        return T.stack([self.pages[:, :, t[i // PAGE], :, i % PAGE] for i in range(n)], 2)


def ints(v):
    return T.tensor(v, dtype=T.int32, device="cuda")


def fork(m, table, lens, parent, new, n_out):
    """(table, lengths, missing) with the copies of all layers done"""
    L, st = m.qa.lib(), T.cuda.current_stream().cuda_stream
    out, ln = T.empty(n_out, m.stride, dtype=T.int32, device="cuda"), T.empty(n_out, dtype=T.int32, device="cuda")
    copies, missing = T.empty(n_out, 4, dtype=T.int32, device="cuda"), T.empty(1, dtype=T.int32, device="cuda")
    kvs = m.kv(table)
    m.qa.check(L.qwen_hip_paged_fork(kvs, lens.data_ptr(), parent.data_ptr(), new.data_ptr(), None, n_out, out.data_ptr(),
                                     ln.data_ptr(), copies.data_ptr(), missing.data_ptr(), None, 0, st), "fork")
    m.qa.check(L.qwen_hip_paged_copy(kvs, m.L, copies.data_ptr(), n_out, st), "copy")
    return out, ln, missing


def select(m, logits, score, ended, seqs, n_out):
    L, (rows, vocab) = m.qa.lib(), logits.shape
    ws = T.empty(L.qwen_hip_beam_select_ws_bytes(seqs, rows // seqs, vocab, n_out), dtype=T.uint8, device="cuda")
    parent, token = (T.empty(seqs * n_out, dtype=T.int32, device="cuda") for _ in range(2))
    out = T.empty(seqs * n_out, device="cuda")
    m.qa.check(L.qwen_hip_beam_select(parent.data_ptr(), token.data_ptr(), out.data_ptr(), logits.data_ptr(), m.qa.ST_F32, vocab,
                                      seqs, rows // seqs, vocab, score.data_ptr(), ended.data_ptr(), n_out, ws.data_ptr(),
                                      ws.numel(), T.cuda.current_stream().cuda_stream), "beam_select")
    return parent, token, out


@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_beam_search(qa, gpu, cache):
    """three sequences of four beams, prompts of 5, 16 and 21 tokens; a beam that draws token 7 is at its end"""
    m, seqs, B = Model(qa, cache, 120, 8), 3, 4
    g = T.Generator().manual_seed(1)
    prompt = [5, 16, 21]
    # the prompts' pages: rows that continue no sequence
    none = T.full((1, m.stride), -1, dtype=T.int32, device="cuda")
    table, lens, missing = fork(m, none, ints([0]), ints([-1] * seqs), ints(prompt), seqs)
    start = ints(np.cumsum([0] + prompt))
    logits = m.rows(T.randint(0, VOCAB, (sum(prompt),), generator=g).cuda(), table, lens, start=start)
    assert int(missing) == 0
    for l in range(m.L):
        m.check_attention(table, prompt, prompt, M.window_sees(2 ** 31 - 1, 0), l)
    logits = logits[[e - 1 for e in start.tolist()[1:]]].contiguous()
    past = [m.cached(table, s, prompt[s]) for s in range(seqs)]
    # the first step: one beam a sequence
    score, ended = T.zeros(seqs, device="cuda"), T.full((seqs,), -1, dtype=T.int32, device="cuda")
    for step in range(12):
        parent, token, best = select(m, logits, score, ended, seqs, B)
        T.cuda.synchronize()
        G.check_beam((parent.view(seqs, B).cpu().numpy(), token.view(seqs, B).cpu().numpy(), best.view(seqs, B).cpu().numpy()),
                     logits, score.tolist(), ended.tolist(), seqs)
        ended = T.where((token == 7) | (ended[parent.long()] >= 0), 7, -1).to(T.int32)
        new = T.ones(seqs * B, dtype=T.int32, device="cuda")
        ref = G.fork_reference(table.tolist(), lens.tolist(), parent.tolist(), [1] * (seqs * B), [], PAGE, m.n_pages)
        table, lens, missing = fork(m, table, lens, parent, new, seqs * B)
        T.cuda.synchronize()
        assert (table.tolist(), lens.tolist(), int(missing)) == (ref[0], ref[1], ref[3])
        logits = m.rows(token, table, lens)
        # every beam's cache is its ancestors' and its own new position
        for s, p in enumerate(parent.tolist()):
            n = int(lens[s])
            now = m.cached(table, s, n)
            assert T.equal(now[:, :, :n - 1], past[p]), (step, s)
        past = [m.cached(table, s, int(lens[s])) for s in range(seqs * B)]
        m.check_attention(table, lens.tolist(), [1] * (seqs * B), M.window_sees(2 ** 31 - 1, 0), step % m.L)
        score = best
    assert len({tuple(r) for r in table.tolist()}) == seqs * B


def greedy(m, tokens, n):
    """n tokens after the prompt, one at a time, and the smallest distance of a largest logit from the next"""
    stride = m.stride
    table = T.arange(stride, dtype=T.int32, device="cuda").view(1, -1)
    got, gap = [], math.inf
    logits = m.rows(tokens, table, ints([len(tokens)]), start=ints([0, len(tokens)]))[-1]
    for i in range(n):
        top = T.topk(logits, 2)[0]
        gap = min(gap, float(top[0] - top[1]))
        got.append(int(logits.argmax()))
        logits = m.rows(ints(got[-1:]), table, ints([len(tokens) + i + 1]))[-1]
    return got, gap


def test_drafts(qa, gpu):
    """a tree of drafts a step: right ones on one branch, wrong ones beside it; the accepted ones move up and the next
    step goes on behind them.  The tokens are those of one step each."""
    m = Model(qa, "f32", 40, 16)
    g = T.Generator().manual_seed(2)
    prompt = T.randint(0, VOCAB, (13,), generator=g)
    want, gap = greedy(m, prompt.cuda(), 40)
    assert gap > 1e-3                                      # far above what the order of sums changes
    m.pages.fill_(math.nan)
    table = T.randperm(40, generator=g)[:16].to(T.int32).view(1, -1).cuda()
    logits = m.rows(prompt.cuda(), table, ints([13]), start=ints([0, 13]))
    have, n, step = [int(logits[-1].argmax())], 13, 0
    while len(have) < 36:
        # the last token, and behind it drafts: each depth two children of the right branch, the right one at either place
        depth = 1 + step % 5
        drafts, parents, right = [have[-1]], [-1], 0
        for d in range(depth):
            true = want[len(have) + d] if d < 1 + step % 4 else -1          # from some depth on no draft is right
            two = [true if true >= 0 else (want[len(have) + d] + 1) % VOCAB, (want[len(have) + d] + 3 + d) % VOCAB]
            if (step + d) % 2:
                two.reverse()
            at = len(drafts)
            drafts += two
            parents += [right, right]
            right = at + (two.index(true) if true >= 0 else 0)
        bits, turn = [], []
        for i, p in enumerate(parents):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
            turn.append(n + bin(bits[i]).count("1") - 1)
        k = len(drafts)
        words = T.tensor(bits, dtype=T.int64, device="cuda").view(-1, 1)
        logits = m.rows(ints(drafts), table, ints([n + k]), start=ints([0, k]), turn=ints(turn), tree=words)
        m.check_attention(table, [n + k], [k], M.tree_sees([bits]), step % m.L)
        said = logits.argmax(-1).tolist()
        path = [0]
        while True:
            nxt = [i for i in range(k) if parents[i] == path[-1] and drafts[i] == said[path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        assert len(path) >= 1 + min(depth, 1 + step % 4)
        before = m.cached(table, 0, n + k)
        ln, kvs = T.zeros(1, dtype=T.int32, device="cuda"), m.kv(table)
        lens, starts, p, c = ints([n + k]), ints([0, k]), ints([path]), ints([len(path)])
        b = qa.PagedBatch(starts.data_ptr(), lens.data_ptr(), k, 0)
        qa.check(qa.lib().qwen_hip_paged_compact(kvs, m.L, C.byref(b), ln.data_ptr(), p.data_ptr(), len(path), c.data_ptr(),
                                                 T.cuda.current_stream().cuda_stream))
        after = m.cached(table, 0, n + len(path))
        assert int(ln) == n + len(path)
        assert T.equal(after[:, :, :n], before[:, :, :n])
        assert T.equal(after[:, :, n:], before[:, :, [n + i for i in path]])
        have += [drafts[i] for i in path[1:]] + [said[path[-1]]]
        n, step = int(ln), step + 1
        assert have == want[:len(have)], step


def test_endless_stream(qa, gpu):
    """a stream of 150 positions that keeps 24 of them and the first 3: pages behind the window are given back and
    taken again, so eight pages are enough; beside it a stream that keeps all"""
    m, win, sinks = Model(qa, "bf16", 28, 20), 24, 3
    g = T.Generator().manual_seed(3)
    table, lens = T.full((2, m.stride), -1, dtype=T.int32, device="cuda"), ints([0, 0])
    most, n = 0, 0
    while n < 150:
        k = [17, 1, 1, 5, 1][n % 5] if n else 20           # pieces and single tokens
        table, lens, missing = fork(m, table, lens, ints([0, 1]), ints([k, k]), 2)
        assert int(missing) == 0
        n += k
        tokens = T.randint(0, VOCAB, (2 * k,), generator=g).cuda()
        # a call for each kind of stream
        for w, rows in (((win, sinks), [0]), ((2 ** 31 - 1, 0), [1])):
            at = [i for r in rows for i in range(r * k, (r + 1) * k)]
            m.rows(tokens[at], table[rows].contiguous(), lens[rows].contiguous(), start=None if k == 1 else ints([0, k]), window=w)
            m.check_attention(table[rows], [n], [k], M.window_sees(*w), n % m.L)
        # what the next row's window does not reach is given back: its ids are -1
        first = n + 1 - win
        for e in range(m.stride):
            if (e + 1) * PAGE <= first and e * PAGE >= sinks:
                table[0, e] = -1
        most = max(most, int((table[0] >= 0).sum()))
    assert most <= 8 and int((table[1] >= 0).sum()) == -(-n // PAGE)


def test_captured_beam_step(qa, gpu):
    """selection, page tables, copies, append and attention of a step captured into a graph, replayed with other scores,
    tokens and tables on the device and eager work between: the same as the eager step, every time"""
    m, seqs, B = Model(qa, "bf16", 64, 6), 2, 3
    g = T.Generator().manual_seed(4)
    n = seqs * B
    none = T.full((1, m.stride), -1, dtype=T.int32, device="cuda")
    t0, l0, _ = fork(m, none, ints([0]), ints([-1] * n), ints([9, 9, 9, 14, 14, 14]), n)
    starts = ints([0, 9, 18, 27, 41, 55, 69])
    m.rows(T.randint(0, VOCAB, (69,), generator=g).cuda(), t0, l0, start=starts)
    T.cuda.synchronize()
    keep = m.pages.clone()
    xs = [(T.randn(n, VOCAB, generator=g).cuda(), -5 * T.rand(n, generator=g).cuda()) for _ in range(3)]
    ended, ones = T.full((n,), -1, dtype=T.int32, device="cuda"), T.ones(n, dtype=T.int32, device="cuda")

    def step(logits, score, table, lens):
        parent, token, best = select(m, logits, score, ended, seqs, B)
        new, ln, missing = fork(m, table, lens, parent, ones, n)
        return parent, token, best, new, ln, missing, m.rows(token, new, ln)

    want = []
    table, lens = t0, l0
    for x, s in xs:
        got = step(x, s, table, lens)
        T.cuda.synchronize()
        want.append([t.clone() for t in got] + [m.pages.clone()])
        table, lens = got[3], got[4]
    side = T.cuda.Stream()
    x, s, table, lens = xs[0][0].clone(), xs[0][1].clone(), t0.clone(), l0.clone()
    T.cuda.synchronize()
    with T.cuda.stream(side):                              # the allocator's blocks of the side stream
        step(x, s, table, lens)
    T.cuda.synchronize()
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        got = step(x, s, table, lens)
    for turn in range(2):
        m.pages.copy_(keep)
        table.copy_(t0), lens.copy_(l0)
        for i in range(3):
            x.copy_(xs[i][0]), s.copy_(xs[i][1])
            graph.replay()
            z = (x * 2.0).sum()                            # eager work between the replays
            T.cuda.synchronize()
            for a, b in zip(list(got) + [m.pages], want[i]):
                assert T.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b), (turn, i)
            table.copy_(got[3]), lens.copy_(got[4])

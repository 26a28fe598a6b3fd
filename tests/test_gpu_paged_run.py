"""The paged cache's operators and the token drawing together, as a program that serves several
streams uses them: packed prompts, then steps of one token each, pages handed out as the streams
grow, the next token drawn from the logits and fed back.  Every operator's result is checked against
its definition in 64 bits on the inputs that the run gave it (tolerances: paged_util, test_gpu_sample)."""
import ctypes as C
import math

import pytest
import torch as T

import paged_util as U
from paged_util import HD
from test_gpu_sample import allowed

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(HD)
EPS = 1e-6


class Server:
    """Streams over one layer's pages: hidden rows -> Q|K|V -> append -> attention -> logits -> tokens"""

    def __init__(self, qa, cache, n, heads=4, kv_heads=2, hidden=256, vocab=1000, page=16, most=8, n_pages=40):
        g = T.Generator().manual_seed(11)
        self.qa, self.cache, self.n, self.H, self.KH, self.page, self.vocab = qa, cache, n, heads, kv_heads, page, vocab
        w = lambda *s: (T.randn(*s, generator=g) * 0.06).bfloat16()
        self.w_qkv, self.w_o, self.emb = w((heads + 2 * kv_heads) * HD, hidden), w(hidden, heads * HD), w(vocab, hidden)
        self.w_head = (T.randn(vocab, hidden, generator=g) * 0.5).bfloat16()
        self.qn, self.kn = (1 + 0.1 * T.randn(HD, generator=g) for _ in range(2))
        self.cos, self.sin = U.rope_tables(most * page)
        self.d = {k: getattr(self, k).cuda() for k in ("w_qkv", "w_o", "emb", "w_head", "qn", "kn", "cos", "sin")}
        shape = (n_pages, kv_heads, page, HD)
        self.k, self.v = (T.full(shape, math.nan, dtype=U.T[cache], device="cuda") for _ in range(2))
        self.table = T.full((n, most), -1, dtype=T.int32)
        self.d_table = self.table.cuda()
        self.lens = [0] * n
        self.free = T.randperm(n_pages, generator=g).tolist()
        self.kv = qa.PagedKV(self.k.data_ptr(), self.v.data_ptr(), self.d_table.data_ptr(),
                             {"f32": qa.ST_F32, "bf16": qa.ST_BF16}[cache], n_pages, page, kv_heads, HD, n, most)

    def grow(self, new):
        """pages for the new rows"""
        for s, k in enumerate(new):
            self.lens[s] += k
            for i in range(-(-self.lens[s] // self.page)):
                if self.table[s, i] < 0:
                    self.table[s, i] = self.free.pop()
        self.d_table.copy_(self.table)
        self.kv_len = T.tensor(self.lens, dtype=T.int32, device="cuda")

    def linear(self, x, w):
        y = T.empty(x.shape[0], w.shape[0], device="cuda")
        self.qa.check(self.qa.lib().qwen_hip_linear_nobias_bf16_noalloc(
            y.data_ptr(), x.data_ptr(), w.data_ptr(), x.shape[0], x.shape[1], w.shape[0],
            T.cuda.current_stream().cuda_stream), "linear")
        return y

    def step(self, x, new, ws):
        """x [rows][hidden] -> (qkv, q after norm and rotation, attention, logits of each stream's last row)"""
        qa, L, H, KH = self.qa, self.qa.lib(), self.H, self.KH
        st = T.cuda.current_stream().cuda_stream
        packed = any(k != 1 for k in new)
        starts = [0]
        for k in new:
            starts.append(starts[-1] + k)
        self.start = T.tensor(starts, dtype=T.int32, device="cuda") if packed else None
        b = qa.PagedBatch(self.start.data_ptr() if packed else None, self.kv_len.data_ptr(), x.shape[0], 0)
        by = C.byref(self.kv), C.byref(b)
        qkv = self.linear(x, self.d["w_qkv"])
        q = T.empty(x.shape[0], H * HD, device="cuda")
        width, at = qkv.shape[1], qkv.data_ptr()
        qa.check(L.qwen_hip_paged_append(*by, q.data_ptr(), at, at + 4 * H * HD, at + 4 * (H + KH) * HD, qa.ST_F32, width,
                                         width, H, self.d["qn"].data_ptr(), self.d["kn"].data_ptr(), EPS,
                                         self.d["cos"].data_ptr(), self.d["sin"].data_ptr(), self.cos.shape[0], st))
        out = T.empty_like(q)
        assert ws.numel() >= L.qwen_hip_paged_attention_ws_bytes(*by, H)
        call = L.qwen_hip_paged_attention_prefill if packed else L.qwen_hip_paged_attention_decode
        qa.check(call(*by, out.data_ptr(), q.data_ptr(), qa.ST_F32, H, SCALE, ws.data_ptr(), ws.numel(), st))
        last = out if not packed else out[[e - 1 for e in starts[1:]]].contiguous()
        h = self.linear(last, self.d["w_o"])
        return qkv, q, out, self.linear(h, self.d["w_head"])

    def draw(self, logits, par, u, ws):
        tokens = T.empty(logits.shape[0], dtype=T.int32, device="cuda")
        p = [t.data_ptr() for t in par]
        self.qa.check(self.qa.lib().qwen_hip_sample(tokens.data_ptr(), logits.data_ptr(), self.vocab, logits.shape[0],
                                                    self.vocab, *p, u.data_ptr(), ws.data_ptr(), ws.numel(),
                                                    T.cuda.current_stream().cuda_stream))
        return tokens


def check_step(S, new, qkv, q, out):
    """append and attention of one step, from the step's own device values"""
    H, KH = S.H, S.KH
    qkv, q, k, v = qkv.cpu(), q.cpu(), S.k.cpu(), S.v.cpu()
    p = U.Paged.__new__(U.Paged)
    p.lens, p.counts, p.group, p.kv_heads, p.heads, p.page = S.lens, new, H // KH, KH, H, S.page
    p.act, p.cache, p.table, p.n_pages, p.rows = "f32", S.cache, S.table, S.k.shape[0], sum(new)
    p.k, p.v, p.q, p.row_start = k, v, q, None
    p.starts = [sum(new[:i]) for i in range(len(new) + 1)]
    for s, (l, c) in enumerate(zip(S.lens, new)):
        for i in range(c):
            row, pos = p.starts[s] + i, l - c + i
            pid = p.page_of(s, pos)
            want = U.norm_rope(qkv[row, :(H + KH) * HD].view(-1, HD), T.cat([S.qn.repeat(H, 1), S.kn.repeat(KH, 1)]), EPS,
                               S.cos[pos], S.sin[pos])
            x = qkv[row, :(H + KH) * HD].view(-1, HD).double()
            # 20 half steps of fp32 of the terms (test_gpu_paged.run_append): both of a pair, at most |w| 1.5
            r = T.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            size = 1.5 * (x.abs() + x.abs().roll(HD // 2, -1)) / r
            tol = 20 * 2.0 ** -24 * size
            assert bool(((q[row].view(H, HD).double() - want[:H]).abs() <= tol[:H] + 2.0 ** -24 * want[:H].abs()).all())
            got = k[pid, :, pos % S.page].double()
            assert bool(((got - want[H:]).abs() <= tol[H:] + U.HALF[S.cache] * want[H:].abs()).all())
            assert T.equal(v[pid, :, pos % S.page], qkv[row, (H + KH) * HD:].view(KH, HD).to(U.T[S.cache]))
    U.check(out, *p.reference(SCALE))


PAR = dict(temperature=[0.0, 0.8, 1.2, 1.0], top_k=[0, 40, 0, 5], top_p=[1.0, 0.9, 0.7, 1.0], min_p=[0.0, 0.02, 0.0, 0.0])


def parameters():
    return [T.tensor(PAR[k], dtype=T.int32 if k == "top_k" else T.float32, device="cuda")
            for k in ("temperature", "top_k", "top_p", "min_p")]


@pytest.mark.parametrize("cache", ["f32", "bf16"])
def test_serving_run(qa, gpu, cache):
    n, g = 4, T.Generator().manual_seed(3)
    S = Server(qa, cache, n)
    ws = T.empty(8 << 20, dtype=T.uint8, device="cuda")
    sws = T.empty(qa.lib().qwen_hip_sample_ws_bytes(n, S.vocab), dtype=T.uint8, device="cuda")
    par = parameters()
    new = [5, 17, 33, 1]
    tokens = T.randint(0, S.vocab, (sum(new),), generator=g)
    produced = []
    for step in range(7):
        S.grow(new)
        x = S.d["emb"].float()[tokens.cuda().long()].contiguous()
        qkv, q, out, logits = S.step(x, new, ws)
        u = T.rand(n, generator=g)
        tok = S.draw(logits, par, u.cuda(), sws)
        T.cuda.synchronize()
        check_step(S, new, qkv, q, out)
        tok, lg = tok.cpu(), logits.cpu().double().numpy()
        for r in range(n):
            one = T.tensor([PAR["temperature"][r], PAR["top_p"][r], PAR["min_p"][r]]).tolist()
            assert int(tok[r]) in allowed(lg[r], one[0], PAR["top_k"][r], one[1], one[2], float(u[r])), (step, r)
        produced.append(tok.tolist())
        tokens, new = tok, [1] * n
    assert len(set(map(tuple, produced))) > 1          # the streams move


def test_captured_step(qa, gpu):
    """a step captured into a graph (append, attention, products, drawing), replayed while lengths, tokens and
    random numbers change on the device, with eager work between: the same bits as the eager step"""
    n = 4
    S = Server(qa, "bf16", n)
    T.cuda.synchronize()
    ws = T.empty(8 << 20, dtype=T.uint8, device="cuda")
    sws = T.empty(qa.lib().qwen_hip_sample_ws_bytes(n, S.vocab), dtype=T.uint8, device="cuda")
    par = parameters()
    new = [20, 7, 33, 2]
    S.grow(new)
    for s in range(n):                                  # room for the steps
        for i in range(4):
            if S.table[s, i] < 0:
                S.table[s, i] = S.free.pop()
    S.d_table.copy_(S.table)
    g = T.Generator().manual_seed(4)
    S.step(T.randn(sum(new), 256, generator=g).cuda(), new, ws)
    T.cuda.synchronize()
    xs = [T.randn(n, 256, generator=g).cuda() for _ in range(4)]
    us = [T.rand(n, generator=g).cuda() for _ in range(4)]
    len0, k0, v0 = S.kv_len.clone(), S.k.clone(), S.v.clone()

    def eager():
        S.kv_len.copy_(len0), S.k.copy_(k0), S.v.copy_(v0)
        got = []
        for x, u in zip(xs, us):
            S.kv_len.add_(1)
            _, _, out, logits = S.step(x, [1] * n, ws)
            got.append((out.clone(), S.draw(logits, par, u, sws).clone()))
            T.cuda.synchronize()
        return got

    want = eager()
    x, u = xs[0].clone(), us[0].clone()
    side = T.cuda.Stream()
    with T.cuda.stream(side):                           # the caching allocator's blocks of the side stream
        S.step(x, [1] * n, ws)
    T.cuda.synchronize()
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        _, _, out, logits = S.step(x, [1] * n, ws)
        tok = S.draw(logits, par, u, sws)
    for _ in range(2):
        S.kv_len.copy_(len0), S.k.copy_(k0), S.v.copy_(v0)
        for i in range(4):
            x.copy_(xs[i]), u.copy_(us[i])
            S.kv_len.add_(1)
            graph.replay()
            z = (x * 2.0).sum()                         # eager work between the replays
            T.cuda.synchronize()
            assert T.equal(out, want[i][0]) and T.equal(tok, want[i][1]), i
    again = eager()
    assert all(T.equal(a, c) and T.equal(b, d) for (a, b), (c, d) in zip(want, again))


def test_two_graphs_with_their_own_workspaces(qa, gpu):
    """two captured attention calls replayed on two streams at once"""
    runs = []
    for i in range(2):
        p = U.Paged(90 + i, [700, 90, 1300], group=2, kv_heads=2, page=16).gpu(qa)
        by = C.byref(p.c_kv), C.byref(p.c_batch)
        need = qa.lib().qwen_hip_paged_attention_ws_bytes(*by, p.heads)
        ws, out = T.empty(need, dtype=T.uint8, device="cuda"), T.zeros_like(p.d["q"])
        T.cuda.synchronize()
        graph, st = T.cuda.CUDAGraph(), T.cuda.Stream()
        with T.cuda.graph(graph, stream=st):
            qa.check(qa.lib().qwen_hip_paged_attention_decode(*by, out.data_ptr(), p.d["q"].data_ptr(), p.c_act, p.heads,
                                                              SCALE, ws.data_ptr(), need, st.cuda_stream))
        runs.append((p, graph, st, out, ws))
    for _ in range(3):
        for p, graph, st, out, ws in runs:
            out.zero_()
        T.cuda.synchronize()
        for _ in range(4):
            for p, graph, st, out, ws in runs:
                with T.cuda.stream(st):
                    graph.replay()
        T.cuda.synchronize()
        for p, graph, st, out, ws in runs:
            U.check(out, *p.reference(SCALE))


def test_same_sequence_twice(qa, gpu):
    """two sequences with the same pages (a shared prefix that neither writes) read the same keys"""
    p = U.Paged(95, [80, 80], group=2, kv_heads=2, page=16)
    p.table[1] = p.table[0]
    p.q[1] = p.q[0]
    out = p.gpu(qa).attention(qa, SCALE)
    assert T.equal(out[0], out[1])
    U.check(out, *p.reference(SCALE))

"""A paged cache with its batch for the tests, and the definitions in 64 bits (CPU, torch.float64)."""
import ctypes as C
import math

import torch

HD = 128
T = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}     # half a rounding step, relative


class Paged:
    """Sequences of `lens` cached positions, the last `new` of them this call's rows (new None: one
    each, no row_start), `front` / `back` rows that belong to no sequence around them.  Everything
    is made on the CPU; gpu() copies it.  Slots that no position uses hold NaN."""

    def __init__(self, seed, lens, new=None, group=2, kv_heads=2, page=16, act="f32", cache="f32", front=0, back=0,
                 spare=3, kstd=1.0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.group, self.kv_heads, self.page = list(lens), new, group, kv_heads, page
        self.act, self.cache, self.front = act, cache, front
        self.heads = group * kv_heads
        n = len(lens)
        self.counts = [1] * n if new is None else list(new)
        self.rows = front + sum(self.counts) + back
        pages = [-(-max(l, 0) // page) for l in lens]
        self.n_pages = sum(pages) + spare
        free = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        self.table = torch.full((n, max(pages + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for s, k in enumerate(pages):
            self.table[s, :k] = free[at:at + k]
            at += k
        shape = (self.n_pages, kv_heads, page, HD)
        self.k = torch.full(shape, math.nan, dtype=T[cache])
        self.v = torch.full(shape, math.nan, dtype=T[cache])
        for s, l in enumerate(lens):
            for p in range(l):
                i = int(self.table[s, p // page])
                self.k[i, :, p % page] = (torch.randn(kv_heads, HD, generator=g) * kstd).to(T[cache])
                self.v[i, :, p % page] = torch.randn(kv_heads, HD, generator=g).to(T[cache])
        self.q = torch.randn(self.rows, self.heads * HD, generator=g).to(T[act])
        starts = [front]
        for c in self.counts:
            starts.append(starts[-1] + c)
        self.starts = starts
        self.kv_len = torch.tensor(lens, dtype=torch.int32)
        self.row_start = None if new is None else torch.tensor(starts, dtype=torch.int32)

    def page_of(self, s, p):
        """page id of position p of sequence s, -1 for none"""
        if p < 0 or p >= self.table.shape[1] * self.page:
            return -1
        i = int(self.table[s, p // self.page])
        return i if 0 <= i < self.n_pages else -1

    def gpu(self, qa, device="cuda"):
        code = {"f32": qa.ST_F32, "bf16": qa.ST_BF16}
        self.d = {n: getattr(self, n).to(device) for n in ("k", "v", "table", "q", "kv_len")}
        if self.row_start is not None:
            self.d["row_start"] = self.row_start.to(device)
        d = self.d
        self.c_kv = qa.PagedKV(d["k"].data_ptr(), d["v"].data_ptr(), d["table"].data_ptr(), code[self.cache],
                               self.n_pages, self.page, self.kv_heads, HD, len(self.lens), self.table.shape[1])
        self.c_batch = qa.PagedBatch(d["row_start"].data_ptr() if self.row_start is not None else None,
                                     d["kv_len"].data_ptr(), self.rows, max(self.lens + [1]))
        self.c_act = code[self.act]
        return self

    def attention(self, qa, scale, max_len=None, stream=None, out=None):
        """the library's result on the device (filled with 7 where it writes nothing)"""
        if max_len is not None:
            self.c_batch.max_len = max_len
        by = C.byref(self.c_kv), C.byref(self.c_batch)
        need = qa.lib().qwen_hip_paged_attention_ws_bytes(*by, self.heads)
        self.ws = torch.full((max(need, 16) // 4,), math.nan, device="cuda")
        if out is None:
            out = torch.full_like(self.d["q"], 7.0)
        call = "decode" if self.row_start is None else "prefill"
        torch.cuda.synchronize()
        rc = getattr(qa.lib(), "qwen_hip_paged_attention_" + call)(
            *by, out.data_ptr(), self.d["q"].data_ptr(), self.c_act, self.heads, scale, self.ws.data_ptr(), need,
            stream)
        qa.check(rc, call)
        torch.cuda.synchronize()
        return out

    def reference(self, scale):
        """(out, tolerance) in 64 bits, a negative tolerance for rows that the call does not write.

        With g(n) = n 2^-24 for a chain of n fp32 operations: a score of 128 products and its
        scaling is off by at most g(136) sum |q_d k_d| scale (the products that a split into
        three bf16 terms drops add 4 2^-24 of it: in the 136), the exponential and its argument
        by 4 2^-24 (1 + |s|) of the weight, the sums over n keys by g(n + 8) of their absolute
        terms each.  bf16 rows of a prefill round each weight by 2^-8, and so do single tokens of more
        than four heads a kv head on a bf16 cache, which run as prompts of one row (all weights of
        an output are rounded, and nothing else is: sum |dw_j v_j| <= 2^-8 sum w_j |v_j|).  The
        result is rounded once more to its type."""
        out = torch.full((self.rows, self.heads, HD), 7.0, dtype=torch.float64)
        tol = torch.full_like(out, -1.0)
        e = 2.0 ** -24
        for s, (l, c) in enumerate(zip(self.lens, self.counts)):
            there = [p for p in range(max(l, 0)) if self.page_of(s, p) >= 0]
            pid = torch.tensor([self.page_of(s, p) for p in there], dtype=torch.int64)
            slot = torch.tensor([p % self.page for p in there], dtype=torch.int64)
            pos = torch.tensor(there)
            k, v = self.k[pid, :, slot].double(), self.v[pid, :, slot].double()     # [n][kv_heads][HD]
            for i in range(c):
                row, p = self.starts[s] + i, max(l, 0) - c + i
                see = pos <= p
                if not bool(see.any()):
                    out[row], tol[row] = 0.0, 0.0
                    continue
                for h in range(self.heads):
                    kk, vv = k[see, h // self.group], v[see, h // self.group]
                    q = self.q[row].view(self.heads, HD)[h].double()
                    sc = kk @ q * scale
                    w = torch.softmax(sc, 0)
                    o = w @ vv
                    n = kk.shape[0]
                    off = 136 * e * (kk.abs() @ q.abs() * scale) + 4 * e * (1 + sc.abs())
                    rel = 2 * off.max() + 2 * (n + 8) * e
                    if self.act == "bf16" and (self.row_start is not None or self.cache == "bf16" and self.group > 4):
                        rel = rel + 2.0 ** -8
                    out[row, h] = o
                    tol[row, h] = 1.1 * (rel * (w @ vv.abs()) + HALF[self.act] * o.abs()) + 1e-37
        return out.view(self.rows, -1), tol.view(self.rows, -1)


def check(got, want, tol):
    """got within tol of want; untouched (7) where tol is negative"""
    got = got.double().cpu()
    left = tol < 0
    assert bool((got[left] == 7.0).all()), "wrote rows that belong to no sequence"
    bad = ~left & ~((got - want).abs() <= tol) & ~(torch.isnan(want) & torch.isnan(got)) & ~(got == want)
    worst = ((got - want).abs() / tol)[~left]
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(worst.nan_to_num(1e9).max()))
    return worst


def rope_tables(n, hd=HD, theta=1e6):
    inv = theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().repeat(1, 2).float(), a.sin().repeat(1, 2).float()


def norm_rope(x, w, eps, cos, sin):
    """[.., HD] in 64 bits; w None: no norm; cos None: no rotation"""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if cos is not None:
        a, b, c, s = x[..., :HD // 2], x[..., HD // 2:], cos.double()[..., :HD // 2], sin.double()[..., :HD // 2]
        x = torch.cat([a * c - b * s, b * c + a * s], -1)
    return x

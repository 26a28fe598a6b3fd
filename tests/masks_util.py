"""Attention of rows that see some of the cache (windows, trees of drafts) for the tests: the definition in
64 bits over paged_util's cache."""
import ctypes as C
import math

import torch

import paged_util as U
from paged_util import HD, HALF


def window_sees(window, sinks):
    return lambda s, i, pos, p, past: (pos <= p) & ((pos > p - window) | (pos < sinks))


def tree_sees(bits):
    """bits[s][i]: the drafts that row i of sequence s sees, a Python integer"""
    def sees(s, i, pos, p, past):
        d = pos - past
        return (pos < past) | torch.tensor([0 <= int(x) and bool(bits[s][i] >> int(x) & 1) for x in d], dtype=torch.bool)
    return sees


def reference(c, scale, sees, matrix):
    """(out, tolerance) of a paged_util.Paged in 64 bits, a negative tolerance for rows of no sequence.

    The bound is paged_util's: a score of 128 products and its scaling is off by at most 136 2^-24
    sum |q_d k_d| scale, the exponential and its argument by 4 2^-24 (1 + |s|), the sums over n
    keys by (n + 8) 2^-24 of their absolute terms each.  On the matrix cores (`matrix`) bf16 rows hold the
    probabilities, and the values of an fp32 cache, in two bf16 terms each: x = h + l + r, where l is
    at most 2^-8 of x and is rounded by at most 2^-8 of itself, so |r| <= 2^-16 |x|; the product l l that is
    left out is at most 2^-16 too: 3 2^-16 in all.  The result is rounded once to its type."""
    out = torch.full((c.rows, c.heads, HD), 7.0, dtype=torch.float64)
    tol = torch.full_like(out, -1.0)
    e = 2.0 ** -24
    for s, (l, n) in enumerate(zip(c.lens, c.counts)):
        there = [p for p in range(min(max(l, 0), c.table.shape[1] * c.page)) if c.page_of(s, p) >= 0]
        pid = torch.tensor([c.page_of(s, p) for p in there], dtype=torch.int64)
        slot = torch.tensor([p % c.page for p in there], dtype=torch.int64)
        pos = torch.tensor(there, dtype=torch.int64)
        k, v = c.k[pid, :, slot].double(), c.v[pid, :, slot].double()
        past = max(l, 0) - n
        for i in range(n):
            row = c.starts[s] + i
            see = sees(s, i, pos, past + i, past)
            if not bool(see.any()):
                out[row], tol[row] = 0.0, 0.0
                continue
            q = c.q[row].view(c.kv_heads, c.group, HD).double()
            kk, vv = k[see].transpose(0, 1), v[see].transpose(0, 1)            # [kv_heads][n][HD]
            sc = q @ kk.transpose(1, 2) * scale
            w = torch.softmax(sc, -1)
            o, size = w @ vv, w @ vv.abs()
            off = 136 * e * (q.abs() @ kk.abs().transpose(1, 2) * scale) + 4 * e * (1 + sc.abs())
            rel = 2 * off.amax(-1, keepdim=True) + 2 * (kk.shape[1] + 8) * e
            if matrix and c.act == "bf16":
                rel = rel + 3 * 2.0 ** -16
            out[row] = o.reshape(c.heads, HD)
            tol[row] = (1.1 * (rel * size + HALF[c.act] * o.abs()) + 1e-37).reshape(c.heads, HD)
    return out.view(c.rows, -1), tol.view(c.rows, -1)


def by_matrix(c):
    return c.row_start is not None or c.cache == "bf16" and c.group > 4


def window(qa, c, scale, win, sinks, max_len=None, stream=None):
    """the library's result on the device (7 where it writes nothing), with a workspace of just the size asked for"""
    if max_len is not None:
        c.c_batch.max_len = max_len
    L, by = qa.lib(), (C.byref(c.c_kv), C.byref(c.c_batch))
    need = L.qwen_hip_paged_attention_window_ws_bytes(*by, c.heads, win, sinks)
    c.ws = torch.full((max(need, 16) // 4,), math.nan, device="cuda")
    out = torch.full_like(c.d["q"], 7.0)
    torch.cuda.synchronize()
    qa.check(L.qwen_hip_paged_attention_window(*by, out.data_ptr(), c.d["q"].data_ptr(), c.c_act, c.heads, scale, win, sinks,
                                               c.ws.data_ptr() if need else None, need, stream), "window")
    torch.cuda.synchronize()
    return out


def tree_words(c, bits, words):
    """[rows][words] of 64 bits as torch holds them; rows of no sequence get ones"""
    t = torch.full((c.rows, words), -1, dtype=torch.int64)
    for s, n in enumerate(c.counts):
        for i in range(n):
            for w in range(words):
                x = bits[s][i] >> (64 * w) & (2 ** 64 - 1)
                t[c.starts[s] + i, w] = x - (x >> 63 << 64)
    return t


def tree(qa, c, scale, bits, words, max_len=None, stream=None):
    if max_len is not None:
        c.c_batch.max_len = max_len
    L, by = qa.lib(), (C.byref(c.c_kv), C.byref(c.c_batch))
    need = L.qwen_hip_paged_attention_tree_ws_bytes(*by, c.heads)
    c.ws = torch.full((max(need, 16) // 4,), math.nan, device="cuda")
    c.tree = tree_words(c, bits, words).cuda()
    out = torch.full_like(c.d["q"], 7.0)
    torch.cuda.synchronize()
    qa.check(L.qwen_hip_paged_attention_tree(*by, out.data_ptr(), c.d["q"].data_ptr(), c.c_act, c.heads, scale,
                                             c.tree.data_ptr(), words, c.ws.data_ptr() if need else None, need, stream), "tree")
    torch.cuda.synchronize()
    return out


def random_tree(g, n, reach=8):
    """ancestors' bits of n drafts, each a child of one of the `reach` before it or of the past"""
    bits = []
    for i in range(n):
        back = int(torch.randint(1, reach + 1, (1,), generator=g))
        bits.append((bits[i - back] if i >= back else 0) | 1 << i)
    return bits

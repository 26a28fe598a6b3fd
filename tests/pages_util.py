"""Definitions of the page tables that continue others and of the choice over beams for the tests (plain Python,
64 bits), and the library's calls on device memory."""
import ctypes as C
import math

import numpy as np
import torch

HD = 128
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def fork_reference(table, lens, parent, new, outside, page, n_pages):
    """(table, lens, copies, missing) as lists"""
    stride = len(table[0])
    n = len(parent)
    ids = lambda p, e: table[p][e] if 0 <= table[p][e] < n_pages else -1
    length = [max(lens[p], 0) if 0 <= p < len(table) else 0 for p in parent]
    kept = [min(-(-l // page), stride) for l in length]
    out = [[ids(p, e) if e < kept[s] else -1 for e in range(stride)] for s, p in enumerate(parent)]
    held = {i for r in out for i in r} | set(outside)
    whole = {out[s][e] for s in range(n) for e in range(min(length[s] // page, stride))} | set(outside)
    inside = [l % page > 0 and l // page < stride for l in length]
    tails = [out[s][length[s] // page] if inside[s] else -1 for s in range(n)]
    free = [i for i in range(n_pages) if i not in held]
    copies, missing = [[-1, -1, 0, 0] for _ in range(n)], 0
    new = [max(k, 0) for k in new]
    fresh = []
    for s in range(n):
        if new[s] == 0:
            continue
        more = any(tails[t] == tails[s] and (length[t] % page, t) > (length[s] % page, s) for t in range(n))
        copied = tails[s] >= 0 and (tails[s] in whole or more)
        first = length[s] // page if inside[s] and (copied or tails[s] < 0) else kept[s]
        need = -(-(length[s] + new[s]) // page)
        missing += max(need - max(stride, -(-length[s] // page)), 0)
        fresh.append((s, copied, range(first, min(need, stride))))
    for s, copied, entries in fresh:
        for j, e in enumerate(entries):
            out[s][e] = free.pop(0) if free else -1
            missing += out[s][e] < 0
            if copied and j == 0 and out[s][e] >= 0:
                copies[s] = [tails[s], out[s][e], 0, length[s] % page]
    return out, [min(l + k, 2 ** 31 - 1) for l, k in zip(length, new)], copies, min(missing, 2 ** 31 - 1)


def fork(qa, table, lens, parent, new, outside, page, n_pages, stream=None):
    ints = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")
    n_in, stride = len(table), len(table[0])
    d = dict(table=ints(table), lens=ints(lens), parent=ints(parent), new=ints(new))
    n = len(parent) if parent is not None else n_in
    hold = None
    if outside:
        hold = torch.zeros(n_pages, dtype=torch.uint8, device="cuda")
        hold[list(outside)] = 1
    kv = qa.PagedKV(None, None, d["table"].data_ptr(), qa.ST_BF16, n_pages, page, 1, HD, n_in, stride)
    out = torch.full((n, stride), 77777, dtype=torch.int32, device="cuda")
    ln, copies, missing = (torch.full(s, 77777, dtype=torch.int32, device="cuda") for s in ((n,), (n, 4), (1,)))
    need = qa.lib().qwen_hip_paged_fork_ws_bytes(C.byref(kv), n)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
    ptr = lambda t: None if t is None else t.data_ptr()
    torch.cuda.synchronize()
    qa.check(qa.lib().qwen_hip_paged_fork(C.byref(kv), ptr(d["lens"]), ptr(d["parent"]), ptr(d["new"]), ptr(hold), n,
                                          ptr(out), ptr(ln), ptr(copies), ptr(missing), ptr(ws) if need else None, need, stream),
             "fork")
    torch.cuda.synchronize()
    return out.tolist(), ln.tolist(), copies.tolist(), int(missing)


def clean(x):
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -math.inf
    return np.minimum(x, float(np.finfo(np.float32).max))


def beam_scores(x, score, ended):
    """[beams][vocab] of one sequence: 64-bit scores, -inf where there is no candidate"""
    x = clean(x)
    out = np.full_like(x, -math.inf)
    for b in range(x.shape[0]):
        s = float(score[b])
        if not math.isfinite(s):
            continue
        if ended is not None and 0 <= ended[b] < x.shape[1]:
            out[b, ended[b]] = s
        elif x[b].max() > -math.inf:
            d = x[b] - x[b].max()
            out[b] = s - math.log(np.exp(d).sum()) + d
    return out


def beam(qa, x, score, ended, n_out, seqs, row_stride=None, stream=None):
    """x [seqs * beams][vocab] tensor on the device (or a view of one with row_stride)"""
    rows, vocab = x.shape
    L, beams = qa.lib(), rows // seqs
    d_score = torch.tensor(score, dtype=torch.float32, device="cuda")
    d_end = None if ended is None else torch.tensor(ended, dtype=torch.int32, device="cuda")
    need = L.qwen_hip_beam_select_ws_bytes(seqs, beams, vocab, n_out)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    parent, token = (torch.full((seqs, n_out), 77777, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.full((seqs, n_out), 7.0, device="cuda")
    torch.cuda.synchronize()
    qa.check(L.qwen_hip_beam_select(parent.data_ptr(), token.data_ptr(), out.data_ptr(), x.data_ptr(),
                                    qa.ST_F32 if x.dtype == torch.float32 else qa.ST_BF16, x.stride(0) if row_stride is None else row_stride,
                                    seqs, beams, vocab, d_score.data_ptr(), None if d_end is None else d_end.data_ptr(), n_out,
                                    ws.data_ptr(), need, stream), "beam_select")
    torch.cuda.synchronize()
    return parent.cpu().numpy(), token.cpu().numpy(), out.cpu().numpy()


# An exponential is off by 1 ulp (2^-23) and by its argument's rounding to fp32 (2^-25): a sum of such by less than 2^-22
# of itself, its logarithm by that.  The score is rounded once more where it is written.
LSE = 2.0 ** -22


def check_beam(got, x, score, ended, seqs):
    """the choice is the definition's: but for scores of two beams nearer than twice LSE, whose order may differ"""
    parent, token, out = got
    x = x.double().cpu().numpy()
    B, n = x.shape[0] // seqs, parent.shape[1]
    for q in range(seqs):
        rows = slice(q * B, (q + 1) * B)
        s = beam_scores(x[rows], score[rows], None if ended is None else ended[rows])
        flat = s.ravel()
        order = np.argsort(-flat, kind="stable")[:n]
        seen = set()
        for k in range(n):
            want = flat[order[k]] if k < len(order) else -math.inf
            if want == -math.inf:
                assert (parent[q, k], token[q, k], out[q, k]) == (-1, -1, -math.inf), (q, k)
                continue
            b, t = int(parent[q, k]) - q * B, int(token[q, k])
            assert 0 <= b < B and 0 <= t < x.shape[1] and (b, t) not in seen, (q, k, b, t)
            seen.add((b, t))
            have = s[b, t]
            assert abs(have - want) <= 2 * LSE, (q, k, have, want)
            assert abs(out[q, k] - have) <= LSE + 2.0 ** -24 * abs(have), (q, k, out[q, k], have)
            same = [j for j in order if j // x.shape[1] == b and flat[j] > -math.inf]
            mine = [int(token[q, j]) for j in range(n) if parent[q, j] == parent[q, k]]
            # in one beam the order is the logits', equal ones by index: no rounding is in it
            assert mine == [int(j % x.shape[1]) for j in np.argsort(-s[b], kind="stable")[:len(mine)]], (q, k)
            assert abs(len(mine) - len(same)) <= 1

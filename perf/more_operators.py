"""The operators a server needs for several continuations of a stream and for streams that do not
end, next to its paged key/value cache (perf/operators.py measures that one):

  window   attention of new rows over a sliding window of the cache and a few first positions
           that stay visible; single tokens (`packed` false) or packed rows
  tree     attention of drafted tokens: a row sees the cached past and its ancestors among the drafts
  compact  the accepted drafts' keys and values move up behind the past, in all layers
  fork     beams that continue chosen beams: page table, pages for the next rows, copies of pages
           that two beams would write, in all layers
  beam     the best continuations over a sequence's beams and the vocabulary

Heads are 128 wide, `group` query heads share a key/value head.  `act` is the type of queries and
outputs (of the logits in `beam`), `cache` the type the pages hold.  A case is a dict of plain
values; `op` selects the operator.  Sequences of one case differ in length: evenly over the
logarithm from `shortest` to `longest`, in an order of their own.
"""
import ctypes
import importlib
import math
import random

import numpy as np
import torch

own = False

HD = 128                       # head size
SCALE = 1.0 / math.sqrt(HD)
VOCAB = 151936
LAYERS = 28
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
INF = math.inf


def listed():
    return [
        # one endless live stream's next token: latency
        {"name": "window_token", "op": "window", "packed": False, "act": "f32", "cache": "f32", "group": 2, "kv_heads": 8,
         "page": 16, "seqs": 1, "longest": 20011, "shortest": 20011, "window": 1024, "sinks": 4},
        # a server's batch of streams of very different ages
        {"name": "window_batch", "op": "window", "packed": False, "act": "bf16", "cache": "bf16", "group": 2,
         "kv_heads": 8, "page": 32, "seqs": 64, "longest": 32769, "shortest": 31, "window": 2048, "sinks": 16},
        # the next pieces of eight recordings behind what they keep, fp32 activations on a bf16 cache
        {"name": "window_chunk", "op": "window", "packed": True, "act": "f32", "cache": "bf16", "group": 2, "kv_heads": 8,
         "page": 64, "seqs": 8, "longest": 515, "shortest": 51, "past": 4000, "window": 1000, "sinks": 17},
        # a long recording's prompt
        {"name": "window_prompt", "op": "window", "packed": True, "act": "bf16", "cache": "bf16", "group": 2,
         "kv_heads": 8, "page": 128, "seqs": 1, "longest": 8191, "shortest": 8191, "past": 0, "window": 1024, "sinks": 64},
        # one live stream's drafts behind a 30 s segment: latency
        {"name": "tree_one", "op": "tree", "act": "f32", "cache": "f32", "group": 2, "kv_heads": 8, "page": 16, "seqs": 1,
         "longest": 16, "shortest": 16, "past": 529},
        # a batch of streams, up to 64 drafts each
        {"name": "tree_batch", "op": "tree", "act": "bf16", "cache": "bf16", "group": 2, "kv_heads": 8, "page": 32,
         "seqs": 24, "longest": 64, "shortest": 21, "past": 4001},
        # what one live stream accepted
        {"name": "compact_one", "op": "compact", "cache": "f32", "kv_heads": 8, "page": 16, "seqs": 1, "longest": 16,
         "shortest": 16, "past": 529, "layers": LAYERS},
        # what a batch of streams accepted
        {"name": "compact_batch", "op": "compact", "cache": "bf16", "kv_heads": 8, "page": 32, "seqs": 24, "longest": 64,
         "shortest": 21, "past": 401, "layers": LAYERS},
        # one stream's four beams take a step
        {"name": "fork_one", "op": "fork", "cache": "f32", "kv_heads": 8, "page": 16, "seqs": 1, "beams": 4, "longest": 530,
         "shortest": 530, "apart": 12, "layers": LAYERS},
        # a batch of streams, eight beams each
        {"name": "fork_batch", "op": "fork", "cache": "bf16", "kv_heads": 8, "page": 32, "seqs": 8, "beams": 8,
         "longest": 701, "shortest": 131, "apart": 40, "layers": LAYERS},
        # one stream's four beams
        {"name": "beam_one", "op": "beam", "act": "f32", "seqs": 1, "beams": 4, "out": 4, "vocab": VOCAB, "spread": 3.0},
        # a batch of streams, eight beams each, twice as many candidates as beams, some beams at their end
        {"name": "beam_batch", "op": "beam", "act": "f32", "seqs": 16, "beams": 8, "out": 16, "vocab": VOCAB, "spread": 2.0},
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["window", "window", "tree", "tree", "compact", "fork", "beam", "beam"])
    if op == "beam":
        beams = log_int(1, 16)
        return {"op": op, "act": rng.choice(["f32", "f32", "bf16"]), "seqs": log_int(1, max(1, 128 // beams)), "beams": beams,
                "out": rng.choice([beams, 2 * beams]), "vocab": rng.choice([VOCAB, log_int(151, 200000)]),
                "spread": rng.choice([0.5, 1.0, 2.0, 3.0, 5.0])}
    act, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
    c = {"op": op, "cache": cache, "kv_heads": rng.choice([1, 2, 4, 8, 8]), "page": rng.choice([16, 32, 64, 128, 256])}
    if op in ("compact", "fork"):
        c["layers"] = rng.choice([LAYERS, log_int(1, LAYERS)])
        row = 2 * SIZE[cache] * HD * c["kv_heads"] * c["layers"]          # bytes of a position
        room = (1 << 30) // row                                           # positions of the pages
        c["seqs"] = log_int(1, min(32, max(1, room // (4 * c["page"] + 256))))
        if op == "compact":
            c["longest"] = log_int(1, 64)
            c["shortest"] = log_int(1, c["longest"])
            c["past"] = log_int(1, max(1, min(2000, room // c["seqs"] - 64 - 2 * c["page"])))
        else:
            c["beams"] = log_int(1, max(1, min(8, room // (c["seqs"] * (2 * c["page"] + 64)))))
            c["apart"] = log_int(1, 64)
            most = room // c["seqs"] - c["beams"] * (3 * c["page"] + c["apart"]) - 4 * c["page"]
            c["longest"] = log_int(2, max(2, min(2000, most)))
            c["shortest"] = log_int(1, c["longest"])
        return c
    c.update(act=act, group=rng.choice([1, 2, 2, 3, 4, 8]))
    heads = c["group"] * c["kv_heads"]
    if op == "tree":
        c["seqs"] = log_int(1, 32)
        c["longest"] = log_int(1, 256)
        c["shortest"] = log_int(1, c["longest"])
        # the plain form holds seqs x heads x longest x (longest + past) scores
        c["past"] = log_int(1, max(1, min(8192, 2 ** 28 // (c["seqs"] * heads * c["longest"]), 2 ** 17 // c["seqs"])))
        return c
    c.update(packed=rng.random() < 0.5, window=log_int(16, 4096), sinks=rng.choice([0, 4, log_int(1, 128)]))
    if not c["packed"]:
        c["seqs"] = log_int(1, 128)
        c["longest"] = log_int(16, 65536)
        c["shortest"] = log_int(1, c["longest"])
        c["window"] = min(c["window"], max(16, (1 << 17) // c["seqs"]))
    else:
        c["seqs"] = log_int(1, 16)
        most = max(64, min(4096, int(math.sqrt(2 ** 28 / (heads * c["seqs"])))))
        c["longest"] = log_int(2, most)
        c["shortest"] = log_int(1, c["longest"])
        room = 2 ** 28 // (heads * c["seqs"] * c["longest"]) - c["longest"] // 2
        c["past"] = rng.choice([0, log_int(1, max(1, min(8192, room)))])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(seqs, shortest, longest):
    """`seqs` lengths from shortest to longest, the same for every seed (they are part of the case)."""
    if seqs == 1:
        return [longest]
    lo, hi = math.log(shortest), math.log(longest)
    got = [int(round(math.exp(lo + (hi - lo) * i / (seqs - 1)))) for i in range(seqs)]
    random.Random(seqs * 7919 + longest).shuffle(got)
    return got


def _shape(case):
    """(new rows, cached positions with the new rows) of each sequence; of a fork: (next rows, cached positions) of each beam"""
    n, past = case["seqs"], case.get("past", 0)
    lens = _lengths(n, case["shortest"], case["longest"])
    if case["op"] == "fork":
        return [1] * (n * case["beams"]), list(np.repeat(lens, case["beams"]))
    if case["op"] == "window" and not case["packed"]:
        return [1] * n, lens
    # pasts differ as well: from a part of it to all of it
    return lens, [a + past * (i + 1) // n for i, a in enumerate(lens)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    t = {"case": case}
    if op == "beam":
        rows, vocab = case["seqs"] * case["beams"], case["vocab"]
        x = _normal(g, rows, vocab, std=case["spread"])
        # tokens the program forbids, and a few likely ones
        x[:, torch.randperm(vocab, generator=g, device="cuda")[: vocab // 100]] = -INF
        x[:, torch.randperm(vocab, generator=g, device="cuda")[:8]] += 2.0 * case["spread"]
        # a beam in eight is at its end: it stays what it is
        end = torch.rand(rows, generator=g, device="cuda") < 0.125
        ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        t.update(logits=x.to(TYPES[case["act"]]), score=-20.0 * torch.rand(rows, generator=g, device="cuda"),
                 ended=torch.where(end, ids, -1).to(torch.int32))
        return t
    rng = np.random.RandomState(int(seed) & 0x7FFFFFFF)
    ps, KH, cache, n = case["page"], case["kv_heads"], TYPES[case["cache"]], case["seqs"]
    new, lens = _shape(case)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    if op == "fork":
        # beams of a sequence share the pages of what they have in common, all but the last `apart` positions
        B = case["beams"]
        pages = [-(-l // ps) for l in lens]
        table, at = np.full((n * B, max(pages) + 2), -1, np.int64), 0
        for s in range(n):
            common = max(0, lens[s * B] - case["apart"]) // ps
            table[s * B:(s + 1) * B, :common] = np.arange(at, at + common)
            at += common
            for b in range(B):
                k = pages[s * B] - common
                table[s * B + b, common:common + k] = np.arange(at, at + k)
                at += k
        n_pages = at + 2 * n * B + 3
        # a sequence's best beams have several continuations
        parent = np.concatenate([np.sort(rng.randint(0, 1 + rng.randint(B), B)) + s * B for s in range(n)])
        t.update(parent=_ints(parent), new_rows=_ints(new))
    else:
        table, at = np.full((n, max(-(-l // ps) for l in lens)), -1, np.int64), 0
        for s in range(n):
            k = -(-lens[s] // ps)
            keep = np.ones(k, bool)
            if op == "window":
                # what no window reaches any more is given back, but for the first positions' pages
                first = lens[s] - new[s] + 1 - case["window"]
                keep = (np.arange(1, k + 1) * ps > first) | (np.arange(k) * ps < case["sinks"])
            table[s, :k][keep] = np.arange(at, at + keep.sum())
            at += int(keep.sum())
        n_pages = at + 3
    # pages are handed out in any order
    order = rng.permutation(n_pages)
    t.update(table=_ints(np.where(table >= 0, order[table], -1)), kv_len=_ints(lens), row_start=_ints(start))
    L = case.get("layers", 1)
    t["pages"] = torch.empty(L, 2, n_pages, KH, ps, HD, dtype=cache, device="cuda").normal_(generator=g)
    if op in ("window", "tree"):
        rows = int(start[-1])
        t["q"] = _normal(g, rows, case["group"] * KH * HD, dtype=TYPES[case["act"]])
        seq = np.repeat(np.arange(n), new)
        t["seq"] = torch.from_numpy(seq).cuda()
        t["pos"] = torch.from_numpy(np.arange(rows) - start[seq] + (np.asarray(lens) - new)[seq]).cuda()
    if op == "tree":
        # a draft continues one of the eight before it (or the past); its bits: itself and its ancestors
        words = -(-max(new) // 64)
        bits = np.zeros((int(start[-1]), words), np.uint64)
        for s in range(n):
            back = rng.randint(1, 9, new[s])
            for i in range(new[s]):
                if i >= back[i]:
                    bits[start[s] + i] = bits[start[s] + i - back[i]]
                bits[start[s] + i, i // 64] |= np.uint64(1 << (i % 64))
        t["tree"] = torch.from_numpy(bits.view(np.int64)).cuda()
    if op == "compact":
        # the accepted drafts in order: a chain of first drafts, then some from behind the accepted ones' places
        path, count = np.zeros((n, max(new)), np.int64), np.zeros(n, np.int64)
        for s in range(n):
            k = rng.randint(0, min(new[s], 12) + 1)
            j = max(rng.randint(0, k + 1), 2 * k - new[s])
            path[s, :j] = np.arange(j)
            path[s, j:k] = np.sort(k + rng.choice(max(new[s] - k, 1), k - j, replace=False))
            count[s] = k
        t.update(path=_ints(path), count=_ints(count))
    return t


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)(state)


def _plain(t):
    case = t["case"]
    if case["op"] == "window" and not case["packed"]:
        return _plain_window_tokens(t)
    return {"window": _plain_rows, "tree": _plain_rows, "compact": _plain_compact, "fork": _plain_fork,
            "beam": _plain_beam}[case["op"]](t)


def _softmax_times(scores, seen, v):
    """softmax over the last axis where `seen`, times v; rows that see nothing are 0"""
    scores = torch.where(seen, scores, -INF)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -INF, 0.0, m))
    l = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(l == 0, 1.0, l)


def _plain_window_tokens(t):
    case = t["case"]
    n, KH, G, ps, sinks = case["seqs"], case["kv_heads"], case["group"], case["page"], case["sinks"]
    # the positions that a token sees: the first ones, and the window's that are not among them
    last = t["kv_len"].long()[:, None]
    pos = torch.arange(-sinks, case["window"], device="cuda").repeat(n, 1)
    pos = torch.where(pos < 0, pos + sinks, last - case["window"] + pos)
    first = torch.arange(pos.shape[1], device="cuda") < sinks
    there = (pos >= 0) & (pos < last) & (first | (pos >= sinks))
    page = t["table"].long().gather(1, (pos // ps).clamp(0, t["table"].shape[1] - 1))
    there &= page >= 0
    k, v = (x[page.clamp_min(0), :, pos % ps].permute(0, 2, 1, 3).float() for x in t["pages"][0])
    v = torch.where(there[:, None, :, None], v, 0.0)
    s = torch.matmul(t["q"].float().view(n, KH, G, HD), k.transpose(2, 3).contiguous()) * SCALE
    return _softmax_times(s, there[:, None, None, :], v).reshape(n, -1).to(t["q"].dtype)


def _plain_rows(t):
    case = t["case"]
    n, KH, G, ps, dt = case["seqs"], case["kv_heads"], case["group"], case["page"], t["q"].dtype
    pos = torch.arange(t["table"].shape[1] * ps, device="cuda")
    page = t["table"][:, pos // ps].long()
    there = (pos < t["kv_len"][:, None]) & (page >= 0)
    k, v = (x[page.clamp_min(0), :, pos % ps].permute(0, 2, 1, 3).float() for x in t["pages"][0])
    v = torch.where(there[:, None, :, None], v, 0.0)
    # packed rows side by side: row i of sequence s at [s][i]
    i = torch.arange(t["pos"].numel(), device="cuda") - t["row_start"].long()[t["seq"]]
    most = int(case["longest"])
    q = torch.zeros(n, most, KH, G, HD, device="cuda")
    at = torch.zeros(n, most, dtype=torch.int64, device="cuda")
    q[t["seq"], i] = t["q"].float().view(-1, KH, G, HD)
    at[t["seq"], i] = t["pos"]
    if case["op"] == "window":
        seen = (pos <= at[..., None]) & ((pos > at[..., None] - case["window"]) | (pos < case["sinks"]))
    else:
        past = (t["kv_len"].long() - t["row_start"].long().diff())[:, None, None]
        words = torch.zeros(n, most, t["tree"].shape[1], dtype=torch.int64, device="cuda")
        words[t["seq"], i] = t["tree"]
        draft = (pos - past).clamp(0, 64 * words.shape[2] - 1).expand(n, most, -1)
        seen = (pos < past) | ((words.gather(2, draft // 64) >> (draft % 64)) & 1).bool()
    seen = (seen & there[:, None])[:, None, :, None]
    q = q.permute(0, 2, 1, 3, 4).reshape(n, KH, most * G, HD)
    s = (torch.matmul(q, k.transpose(2, 3).contiguous()) * SCALE).view(n, KH, most, G, -1)
    s = torch.where(seen, s, -INF).view(n, KH, most * G, -1)
    o = _softmax_times(s, there[:, None, None, :], v)
    o = o.view(n, KH, most, G, HD).permute(0, 2, 1, 3, 4)[t["seq"], i]
    return o.reshape(o.shape[0], -1).to(dt)


def _plain_compact(t):
    ps = t["case"]["page"]
    past = t["kv_len"].long() - t["row_start"].long().diff()
    i = torch.arange(t["path"].shape[1], device="cuda")
    seq, at = torch.nonzero(i < t["count"][:, None], as_tuple=True)
    to, frm = past[seq] + at, past[seq] + t["path"].long()[seq, at]
    page = t["table"].long()
    rows = t["pages"][:, :, page[seq, frm // ps], :, frm % ps]
    t["pages"][:, :, page[seq, to // ps], :, to % ps] = rows
    return [t["pages"], (past + t["count"]).to(torch.int32)]


def _plain_fork(t):
    ps, n_pages, stride = t["case"]["page"], t["pages"].shape[2], t["table"].shape[1]
    parent = t["parent"].long()
    length = torch.where(parent >= 0, t["kv_len"].long()[parent.clamp_min(0)], 0)
    new_len = length + t["new_rows"]
    e = torch.arange(stride, device="cuda")
    table = torch.where(e < -(-length // ps)[:, None], t["table"].long()[parent.clamp_min(0)], -1)
    held = torch.zeros(n_pages + 1, dtype=torch.bool, device="cuda")
    held[torch.where(table >= 0, table, n_pages)] = True
    whole = torch.zeros_like(held)
    whole[torch.where((table >= 0) & (e < (length // ps)[:, None]), table, n_pages)] = True
    # a last page with room that another beam holds too is copied, but for the last beam that holds it
    part = length % ps
    tail = table.gather(1, (length // ps).clamp_max(stride - 1)[:, None])[:, 0]
    tail = torch.where(part > 0, tail, -1)
    later = ((tail[:, None] == tail) & (tail >= 0)[:, None]).triu(1).any(1)
    writes = (part > 0) & (t["new_rows"] > 0)
    copied = writes & (tail >= 0) & (later | whole[tail.clamp_min(0)])
    fresh = (e >= -(-length // ps)[:, None]) & (e < -(-new_len // ps)[:, None])
    fresh |= (e == (length // ps)[:, None]) & (writes & (copied | (tail < 0)))[:, None]
    row, entry = torch.nonzero(fresh, as_tuple=True)
    ids = torch.nonzero(~held[:n_pages])[: row.numel(), 0]
    table[row, entry] = ids
    to = table.gather(1, (length // ps).clamp_max(stride - 1)[:, None])[:, 0]
    zero = torch.zeros_like(tail)
    copies = torch.stack([torch.where(copied, tail, -1), torch.where(copied, to, -1), zero, torch.where(copied, part, zero)], 1)
    # the copied slots in all layers
    row, slot = torch.nonzero(copied[:, None] & (torch.arange(ps, device="cuda") < part[:, None]), as_tuple=True)
    t["pages"][:, :, to[row], :, slot] = t["pages"][:, :, tail[row], :, slot]
    return [t["pages"]] + [x.to(torch.int32) for x in (table, new_len, copies)]


def _plain_beam(t):
    case = t["case"]
    n, B, vocab, k = case["seqs"], case["beams"], case["vocab"], case["out"]
    # 64 bits: candidates next to each other in different beams
    x = t["logits"].double()
    m = x.amax(-1, keepdim=True)
    x = x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))) + t["score"].double()[:, None]
    end = t["ended"].long()[:, None]
    stays = torch.where(torch.arange(vocab, device="cuda") == end, t["score"].double()[:, None], -INF)
    x = torch.where(end >= 0, stays, x).view(n, B * vocab)
    best, at = torch.sort(x, dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    none = best == -INF
    parent = at // vocab + B * torch.arange(n, device="cuda")[:, None]
    return [torch.where(none, -1, parent).to(torch.int32), torch.where(none, -1, at % vocab).to(torch.int32), best.float()]


def _own(t):
    QA = t.get("QA")
    if QA is None:
        # a program's handles, kept from call to call: the cache's descriptors, the batch's, a workspace
        QA = t["QA"] = importlib.import_module("qwen-asr_amd")
        t["need"] = _own_handles(t, QA, QA.lib())
        t["ws"] = torch.empty(max(t["need"], 16), dtype=torch.uint8, device="cuda")
    L, case, s = QA.lib(), t["case"], torch.cuda.current_stream().cuda_stream
    op, ws = case["op"], (t["ws"].data_ptr(), t["ws"].numel(), s)
    ptr = lambda name: t[name].data_ptr()
    if op == "beam":
        n, k = case["seqs"], case["out"]
        ids, score = torch.empty(2, n, k, dtype=torch.int32, device="cuda"), torch.empty(n, k, device="cuda")
        parent, token = ids
        QA.check(L.qwen_hip_beam_select(parent.data_ptr(), token.data_ptr(), score.data_ptr(), ptr("logits"), t["act"],
                                        case["vocab"], n, case["beams"], case["vocab"], ptr("score"), ptr("ended"), k, *ws),
                 "beam_select")
        return [parent, token, score]
    if op == "compact":
        lens = torch.empty_like(t["kv_len"])
        QA.check(L.qwen_hip_paged_compact(t["layers"], case["layers"], t["batch"], lens.data_ptr(), ptr("path"),
                                          t["path"].shape[1], ptr("count"), s), "paged_compact")
        return [t["pages"], lens]
    if op == "fork":
        rows = t["parent"].numel()
        table, lens = torch.empty_like(t["table"]), torch.empty_like(t["parent"])
        copies = torch.empty(rows, 4, dtype=torch.int32, device="cuda")
        QA.check(L.qwen_hip_paged_fork(t["layers"], ptr("kv_len"), ptr("parent"), ptr("new_rows"), None, rows,
                                       table.data_ptr(), lens.data_ptr(), copies.data_ptr(), ptr("missing"), *ws), "paged_fork")
        QA.check(L.qwen_hip_paged_copy(t["layers"], case["layers"], copies.data_ptr(), rows, s), "paged_copy")
        return [t["pages"], table, lens, copies]
    out = torch.empty_like(t["q"])
    H = case["group"] * case["kv_heads"]
    if op == "window":
        QA.check(L.qwen_hip_paged_attention_window(t["layers"], t["batch"], out.data_ptr(), ptr("q"), t["act"], H, SCALE,
                                                   case["window"], case["sinks"], *ws), "window")
    else:
        QA.check(L.qwen_hip_paged_attention_tree(t["layers"], t["batch"], out.data_ptr(), ptr("q"), t["act"], H, SCALE,
                                                 ptr("tree"), t["tree"].shape[1], *ws), "tree")
    return out


def _own_handles(t, QA, L):
    """the handles of a state, and the bytes of its workspace"""
    case = t["case"]
    code = {"f32": QA.ST_F32, "bf16": QA.ST_BF16}
    t["act"] = code[case.get("act", "f32")]
    if case["op"] == "beam":
        return L.qwen_hip_beam_select_ws_bytes(case["seqs"], case["beams"], case["vocab"], case["out"])
    n, stride = t["table"].shape
    layers = [QA.PagedKV(p[0].data_ptr(), p[1].data_ptr(), t["table"].data_ptr(), code[case["cache"]], p.shape[1], case["page"],
                         case["kv_heads"], HD, n, stride) for p in t["pages"]]
    t["layers"] = (QA.PagedKV * len(layers))(*layers)
    if case["op"] == "fork":
        t["missing"] = torch.empty(1, dtype=torch.int32, device="cuda")
        return L.qwen_hip_paged_fork_ws_bytes(t["layers"], t["parent"].numel())
    packed = case.get("packed", True)
    new, lens = _shape(case)
    batch = QA.PagedBatch(t["row_start"].data_ptr() if packed else None, t["kv_len"].data_ptr(), sum(new), max(lens))
    t["batch"] = ctypes.byref(batch)
    if case["op"] == "compact":
        return 0
    H = case["group"] * case["kv_heads"]
    if case["op"] == "tree":
        return L.qwen_hip_paged_attention_tree_ws_bytes(t["layers"], t["batch"], H)
    return L.qwen_hip_paged_attention_window_ws_bytes(t["layers"], t["batch"], H, case["window"], case["sinks"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "beam":
        rows = case["seqs"] * case["beams"]
        # a comparison, an exponential and a sum for each entry
        return {"bytes": float(rows * (SIZE[case["act"]] * case["vocab"] + 8) + 12 * case["seqs"] * case["out"]),
                "flops": 4.0 * rows * case["vocab"]}
    new, lens = _shape(case)
    KH, c, ps, n = case["kv_heads"], SIZE[case["cache"]], case["page"], case["seqs"]
    if case["op"] == "compact":
        # half of the up to twelve accepted drafts move, read once and written once
        moved = sum(min(m, 12) / 4 for m in new)
        return {"bytes": moved * 4 * c * KH * HD * case["layers"] + 12.0 * n, "flops": 0.0}
    if case["op"] == "fork":
        # a third of the beams, about, copies its last page's rows; the table is read and written
        moved = sum(l % ps for l in lens) / 3
        return {"bytes": moved * 4 * c * KH * HD * case["layers"] + 8.0 * sum(-(-l // ps) for l in lens), "flops": 0.0}
    a, G = SIZE[case["act"]], case["group"]
    rows = 2 * a * sum(new) * G * KH * HD
    if case["op"] == "tree":
        # past and half of the drafts
        pairs = sum(m * (l - m) + m * m / 2 for m, l in zip(new, lens))
        return {"bytes": float(rows + 2 * c * KH * HD * sum(lens) + 8 * sum(new) * -(-max(new) // 64)),
                "flops": 4.0 * HD * G * KH * pairs}
    W, S = case["window"], case["sinks"]
    # keys of a row at position p: the window's and the first ones that it does not hold
    keys = lambda p: np.minimum(p + 1, W) + np.clip(p + 1 - W, 0, S)
    pairs = float(sum(keys(np.arange(l - m, l)).sum() for m, l in zip(new, lens)))
    seen = sum(min(l, m - 1 + W + min(S, max(0, l - m + 1 - W))) for m, l in zip(new, lens))
    return {"bytes": float(rows + 2 * c * KH * HD * seen), "flops": 4.0 * HD * G * KH * pairs}


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def exact(case, seed):
    t = prepare(case, seed)
    op, n = case["op"], case["seqs"]
    if op == "beam":
        B, vocab, got = case["beams"], case["vocab"], []
        for s in range(n):
            found = []
            for b in range(s * B, (s + 1) * B):
                x, score, end = t["logits"][b].double().cpu().numpy(), float(t["score"][b]), int(t["ended"][b])
                if end >= 0:
                    found.append((-score, b, end))
                    continue
                top = np.argsort(-x, kind="stable")[: case["out"]]
                lse = np.logaddexp.reduce(x[np.isfinite(x)])
                found += [(-(score + float(x[i] - lse)), b, int(i)) for i in top if x[i] > -INF]
            found = sorted(found)[: case["out"]]
            got.append(found + [(INF, -1, -1)] * (case["out"] - len(found)))
        got = np.array(got)
        return [got[..., 1].astype(np.int32), got[..., 2].astype(np.int32), -got[..., 0]]
    new, lens = _shape(case)
    KH, ps, table = case["kv_heads"], case["page"], t["table"].long().cpu().numpy()
    if op == "compact":
        done = t["pages"].clone()
        count, path = t["count"].tolist(), t["path"].tolist()
        for s in range(n):
            for i in range(count[s]):
                a, b = lens[s] - new[s] + i, lens[s] - new[s] + path[s][i]
                done[:, :, table[s, a // ps], :, a % ps] = t["pages"][:, :, table[s, b // ps], :, b % ps]
        return [done, np.array([l - m + k for l, m, k in zip(lens, new, count)], np.int32)]
    if op == "fork":
        done, parent, rows = t["pages"].clone(), t["parent"].tolist(), len(lens)
        length = [lens[p] for p in parent]
        out = np.full_like(table, -1)
        for s in range(rows):
            k = -(-length[s] // ps)
            out[s, :k] = table[parent[s], :k]
        free = sorted(set(range(t["pages"].shape[2])) - set(out.ravel().tolist()))
        kept, copies = out.copy(), []
        for s in range(rows):
            e, part = length[s] // ps, length[s] % ps
            copies.append([-1, -1, 0, 0])
            if part == 0:
                out[s, e] = free.pop(0)
                continue
            mine = kept[s, e]
            holders = [(r, x) for r in range(rows) for x in np.flatnonzero(kept[r] == mine)]
            if any(r > s or x < length[r] // ps for r, x in holders):
                out[s, e] = free.pop(0)
                copies[-1] = [mine, out[s, e], 0, part]
                done[:, :, out[s, e], :, :part] = t["pages"][:, :, mine, :, :part]
        return [done, out.astype(np.int32), np.array([l + 1 for l in length], np.int32), np.array(copies, np.int32)]
    G, outs, at = case["group"], [], 0
    for s, (m, l) in enumerate(zip(new, lens)):
        pos, p = np.arange(l), np.arange(l - m, l)[:, None]
        if op == "window":
            see = (pos <= p) & ((pos > p - case["window"]) | (pos < case["sinks"]))
        else:
            bits = t["tree"][at:at + m].cpu().numpy().view(np.uint64)
            drafts = np.unpackbits(bits.view(np.uint8), axis=1, bitorder="little")[:, :m].astype(bool)
            see = np.concatenate([np.ones((m, l - m), bool), drafts], 1)
        use = np.flatnonzero(see.any(0))                   # pages of the others may be gone
        mask = torch.from_numpy(see[:, use]).cuda()
        ids, slot = (torch.from_numpy(x).cuda() for x in (table[s, use // ps], use % ps))
        k, v = (x[ids, :, slot].double().transpose(0, 1) for x in t["pages"][0])
        q = t["q"][at:at + m].double().view(m, KH, G, HD)
        heads = [torch.softmax((q[:, h, g] @ k[h].t() / math.sqrt(HD)).masked_fill(~mask, -INF), -1) @ v[h]
                 for h in range(KH) for g in range(G)]
        outs.append(torch.cat(heads, 1))
        at += m
    return torch.cat(outs)

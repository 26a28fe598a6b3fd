"""The operators a server of several audio streams needs next to the decoder: a
paged key/value cache, the attention that reads it, and drawing tokens.

Heads are 128 wide (the decoder's only head size), `group` query heads share a
key/value head.  `act` is the type of the queries, keys, values and outputs that
go through the call, `cache` the type the pages hold.  A case is a dict of plain
values; `op` selects the operator:

  append   RMS norm and rotation of new rows' queries and keys, keys and values
           stored into the pages
  decode   attention of one new row per sequence over its pages
  prefill  causal attention of packed prompts (each on top of its cached past)
           over their pages
  sample   temperature, top-k, top-p, min-p, then a draw at a given random number

Sequences of one case differ in length: their lengths lie between `shortest` and
`longest` (evenly over the logarithm, in an order of their own).
"""
import ctypes
import importlib
import math
import random

import numpy as np
import torch

own = False

HD = 128                       # head size
EPS, THETA = 1e-6, 1e6
SCALE = 1.0 / math.sqrt(HD)
VOCAB = 151936
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


def listed():
    return [
        # one live stream's next token enters the cache: launch latency
        {"name": "append_token", "op": "append", "act": "f32", "cache": "f32", "group": 2, "kv_heads": 8, "page": 16,
         "seqs": 1, "new_longest": 1, "new_shortest": 1, "past": 529},
        # the prompts of eight recordings of up to two minutes, norms and rotation applied on the way
        {"name": "append_prompts", "op": "append", "act": "bf16", "cache": "bf16", "group": 2, "kv_heads": 8,
         "page": 64, "seqs": 8, "new_longest": 1515, "new_shortest": 101, "past": 26},
        # one live stream, a 30 s segment in the cache: latency
        {"name": "decode_one", "op": "decode", "act": "f32", "cache": "f32", "group": 2, "kv_heads": 8, "page": 16,
         "seqs": 1, "longest": 530, "shortest": 530},
        # a server's batch of streams of very different ages
        {"name": "decode_batch", "op": "decode", "act": "bf16", "cache": "bf16", "group": 2, "kv_heads": 8,
         "page": 32, "seqs": 64, "longest": 4097, "shortest": 31},
        # a few hour-long recordings on fp32 activations and a cache of half the size
        {"name": "decode_long", "op": "decode", "act": "f32", "cache": "bf16", "group": 4, "kv_heads": 8, "page": 256,
         "seqs": 3, "longest": 32769, "shortest": 20011},
        # a live stream's next chunk behind the prefix that it keeps
        {"name": "prefill_chunk", "op": "prefill", "act": "f32", "cache": "f32", "group": 2, "kv_heads": 8,
         "page": 16, "seqs": 1, "longest": 31, "shortest": 31, "past": 993},
        # eight recordings' prompts at once, fp32 activations on a bf16 cache
        {"name": "prefill_packed", "op": "prefill", "act": "f32", "cache": "bf16", "group": 2, "kv_heads": 8,
         "page": 64, "seqs": 8, "longest": 1515, "shortest": 101, "past": 0},
        # a long recording's prompt
        {"name": "prefill_long", "op": "prefill", "act": "bf16", "cache": "bf16", "group": 2, "kv_heads": 8,
         "page": 128, "seqs": 1, "longest": 8191, "shortest": 8191, "past": 0},
        # one stream's answer: every filter on
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": VOCAB, "mode": "all", "spread": 3.0},
        # a batch of streams, the nucleus alone
        {"name": "sample_batch", "op": "sample", "rows": 64, "vocab": VOCAB, "mode": "top_p", "spread": 2.0},
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "sample"])
    if op == "sample":
        rows, vocab = log_int(1, 96), rng.choice([VOCAB, log_int(151, 200000)])
        return {"op": op, "rows": rows, "vocab": vocab, "spread": rng.choice([0.5, 1.0, 2.0, 3.0, 5.0]),
                "mode": rng.choice(["none", "top_k", "top_p", "min_p", "all"])}
    act, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
    c = {"op": op, "act": act, "cache": cache, "group": rng.choice([1, 2, 2, 3, 4, 8]),
         "kv_heads": rng.choice([1, 2, 4, 8, 8]), "page": rng.choice([16, 32, 64, 128, 256])}
    heads = c["group"] * c["kv_heads"]
    if op == "append":
        c["seqs"] = log_int(1, 64)
        c["new_longest"] = 1 if rng.random() < 0.3 else log_int(2, max(2, 16384 // c["seqs"]))
        c["new_shortest"] = log_int(1, c["new_longest"])
        c["past"] = log_int(1, 2048)
    elif op == "decode":
        c["seqs"] = log_int(1, 128)
        c["longest"] = log_int(16, max(16, min(32768, (1 << 18) // c["seqs"])))
        c["shortest"] = log_int(1, c["longest"])
    else:
        # the plain form holds seqs x heads x longest x (longest + past) scores
        c["seqs"] = log_int(1, 16)
        most = max(64, min(4096, int(math.sqrt(2 ** 29 / (heads * c["seqs"])))))
        c["longest"] = log_int(2, most)
        c["shortest"] = log_int(1, c["longest"])
        # no more products than the longest prompt above has
        room = 2 ** 29 // (heads * c["seqs"] * c["longest"]) - c["longest"] // 2
        c["past"] = rng.choice([0, log_int(1, max(1, min(8192, room)))])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(seqs, shortest, longest):
    """`seqs` lengths from shortest to longest, the same for every seed (they are part of the case)."""
    if seqs == 1:
        return [longest]
    got = [int(round(math.exp(math.log(shortest) + (math.log(longest) - math.log(shortest)) * i / (seqs - 1))))
           for i in range(seqs)]
    random.Random(seqs * 7919 + longest).shuffle(got)
    return got


def _shape(case):
    """(new rows, cached positions with the new rows) of each sequence"""
    n, past = case["seqs"], case.get("past", 0)
    if case["op"] == "append":
        new = _lengths(n, case["new_shortest"], case["new_longest"])
    elif case["op"] == "prefill":
        new = _lengths(n, case["shortest"], case["longest"])
    else:
        return [1] * n, _lengths(n, case["shortest"], case["longest"])
    # pasts differ as well: from none of it to all of it
    pasts = [past * (i + 1) // n for i in range(n)]
    return new, [a + b for a, b in zip(new, pasts)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _sample_inputs(case, seed):
    g, rows, vocab, mode = _gen(seed), case["rows"], case["vocab"], case["mode"]
    logits = _normal(g, rows, vocab, std=case["spread"])
    # tokens the program forbids
    logits[:, torch.randperm(vocab, generator=g, device="cuda")[: vocab // 100]] = -math.inf
    # a few likely ones, as a model's answer has them
    logits[:, torch.randperm(vocab, generator=g, device="cuda")[:8]] += 2.0 * case["spread"]
    uni = lambda lo, hi: torch.rand(rows, generator=g, device="cuda") * (hi - lo) + lo
    on = lambda *m: mode in m or mode == "all"
    top_k = torch.randint(1, max(2, min(vocab, 400)), (rows,), generator=g, device="cuda", dtype=torch.int32)
    return {"logits": logits, "temperature": uni(0.6, 1.3), "u": torch.rand(rows, generator=g, device="cuda"),
            "top_k": top_k if on("top_k") else torch.zeros_like(top_k),
            "top_p": uni(0.5, 0.98) if on("top_p") else torch.ones(rows, device="cuda"),
            "min_p": uni(0.01, 0.2) if on("min_p") else torch.zeros(rows, device="cuda")}


def _paged_inputs(case, seed):
    g, ps, KH = _gen(seed), case["page"], case["kv_heads"]
    H, act, cache = case["group"] * KH, TYPES[case["act"]], TYPES[case["cache"]]
    new, lens = _shape(case)
    n, rows = case["seqs"], sum(new)
    pages = [-(-l // ps) for l in lens]
    n_pages = sum(pages) + 3
    # pages are handed out in any order
    free = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n, max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, k in enumerate(pages):
        table[s, :k] = free[at:at + k]
        at += k
    start = np.concatenate([[0], np.cumsum(new)])
    ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")
    t = {"k_pages": _normal(g, n_pages, KH, ps, HD, dtype=cache), "v_pages": _normal(g, n_pages, KH, ps, HD, dtype=cache),
         "table": table, "kv_len": ints(lens), "row_start": ints(start)}
    # where each packed row comes from: its sequence and its position there
    seq = np.repeat(np.arange(n), new)
    t["seq"] = torch.from_numpy(seq).cuda()
    t["pos"] = torch.from_numpy(np.arange(rows) - start[seq] + (np.asarray(lens) - new)[seq]).cuda()
    if case["op"] == "append":
        inv = 1.0 / THETA ** (torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
        ang = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * inv
        t.update(q=_normal(g, rows, H * HD, dtype=act), k=_normal(g, rows, KH * HD, dtype=act),
                 v=_normal(g, rows, KH * HD, dtype=act), q_norm=_normal(g, HD, std=0.1, mean=1.0),
                 k_norm=_normal(g, HD, std=0.1, mean=1.0),
                 cos=ang.cos().repeat(1, 2).float(), sin=ang.sin().repeat(1, 2).float())
    else:
        t["q"] = _normal(g, rows, H * HD, dtype=act)
    return t


def prepare(case, seed):
    t = _sample_inputs(case, seed) if case["op"] == "sample" else _paged_inputs(case, seed)
    t["case"] = case
    return t


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)(state)


def _plain(t):
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
            "sample": _plain_sample}[t["case"]["op"]](t)


def _plain_append(t):
    case = t["case"]
    KH, ps = case["kv_heads"], case["page"]
    cos, sin = t["cos"][t["pos"]][:, None, :HD // 2], t["sin"][t["pos"]][:, None, :HD // 2]

    def rotated(x, w):
        x = x.float().view(x.shape[0], -1, HD)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :HD // 2], x[..., HD // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    page = t["table"][t["seq"], t["pos"] // ps].long()
    slot = t["pos"] % ps
    t["k_pages"][page, :, slot] = rotated(t["k"], t["k_norm"]).to(t["k_pages"].dtype)
    t["v_pages"][page, :, slot] = t["v"].float().view(-1, KH, HD).to(t["v_pages"].dtype)
    return [rotated(t["q"], t["q_norm"]).flatten(1).to(t["q"].dtype), t["k_pages"], t["v_pages"]]


def _gathered(t):
    """the sequences' keys and values [seqs][kv_heads][longest][HD] in 32 bits, and which are there"""
    ps, longest = t["case"]["page"], t["table"].shape[1] * t["case"]["page"]
    pos = torch.arange(longest, device="cuda")
    page = t["table"][:, pos // ps].long().clamp_min(0)
    there = pos < t["kv_len"][:, None]
    k, v = (x[page, :, pos % ps].permute(0, 2, 1, 3).float() for x in (t["k_pages"], t["v_pages"]))
    return k.contiguous(), torch.where(there[:, None, :, None], v, 0.0).contiguous(), there


def _softmax_times(scores, seen, v):
    """softmax over the last axis where `seen`, times v"""
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _plain_decode(t):
    case = t["case"]
    n, KH, G = case["seqs"], case["kv_heads"], case["group"]
    k, v, there = _gathered(t)
    q = t["q"].float().view(n, KH, G, HD)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * SCALE
    return _softmax_times(s, there[:, None, None, :], v).reshape(n, -1).to(t["q"].dtype)


def _plain_prefill(t):
    case = t["case"]
    n, KH, G, dt = case["seqs"], case["kv_heads"], case["group"], t["q"].dtype
    k, v, there = _gathered(t)
    # packed rows side by side: row i of sequence s at [s][i]
    i = torch.arange(t["pos"].numel(), device="cuda") - t["row_start"].long()[t["seq"]]
    most = int(case["longest"])
    q = torch.zeros(n, most, KH, G, HD, device="cuda")
    at = torch.zeros(n, most, dtype=torch.int64, device="cuda")
    q[t["seq"], i] = t["q"].float().view(-1, KH, G, HD)
    at[t["seq"], i] = t["pos"]
    q = q.permute(0, 2, 1, 3, 4).reshape(n, KH, most * G, HD)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * SCALE
    s = s.view(n, KH, most, G, -1)
    seen = torch.arange(k.shape[2], device="cuda") <= at[..., None]
    s = torch.where(seen[:, None, :, None, :], s, -math.inf)
    o = _softmax_times(s.view(n, KH, most * G, -1), there[:, None, None, :], v)
    o = o.view(n, KH, most, G, HD).permute(0, 2, 1, 3, 4)[t["seq"], i]
    return o.reshape(o.shape[0], -1).to(dt)


def _plain_sample(t):
    vocab = t["case"]["vocab"]
    # 64 bits: a draw at the border of two tokens
    x = t["logits"].double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / t["temperature"].double()[:, None])
    ranked, order = torch.sort(w, dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(t["top_k"] > 0, t["top_k"].long(), vocab)[:, None]
    ranked = torch.where(rank < k, ranked, 0.0)
    before = ranked.cumsum(-1) - ranked
    p = t["top_p"].double()[:, None]
    keep = (rank < k) & ((before < p * ranked.sum(-1, keepdim=True)) | (p >= 1))
    keep &= ranked >= t["min_p"].double()[:, None]
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0.0))
    cdf = kept.cumsum(-1)
    return (cdf <= t["u"].double()[:, None] * cdf[:, -1:]).sum(-1).to(torch.int32)


def _own(t):
    QA = t.get("QA")
    if QA is None:
        # a program's handles, kept from call to call: the cache's descriptor, the batch's, a workspace
        QA = t["QA"] = importlib.import_module("qwen-asr_amd")
        case = t["case"]
        if case["op"] == "sample":
            n = QA.lib().qwen_hip_sample_ws_bytes(case["rows"], case["vocab"])
        else:
            KH, n_pages = case["kv_heads"], t["k_pages"].shape[0]
            code = {"f32": QA.ST_F32, "bf16": QA.ST_BF16}
            t["act"] = code[case["act"]]
            t["kv"] = QA.PagedKV(t["k_pages"].data_ptr(), t["v_pages"].data_ptr(), t["table"].data_ptr(),
                                 code[case["cache"]], n_pages, case["page"], KH, HD, case["seqs"], t["table"].shape[1])
            t["batch"] = QA.PagedBatch(None if case["op"] == "decode" else t["row_start"].data_ptr(),
                                       t["kv_len"].data_ptr(), t["q"].shape[0], max(_shape(case)[1]))
            t["by"] = ctypes.byref(t["kv"]), ctypes.byref(t["batch"])
            n = QA.lib().qwen_hip_paged_attention_ws_bytes(*t["by"], case["group"] * KH)
        t["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    L, case, s = QA.lib(), t["case"], torch.cuda.current_stream().cuda_stream
    ptr = lambda name: t[name].data_ptr()
    if case["op"] == "sample":
        tokens = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        QA.check(L.qwen_hip_sample(tokens.data_ptr(), ptr("logits"), case["vocab"], case["rows"], case["vocab"],
                                   ptr("temperature"), ptr("top_k"), ptr("top_p"), ptr("min_p"), ptr("u"), ptr("ws"),
                                   t["ws"].numel(), s), "sample")
        return tokens
    H, KH = case["group"] * case["kv_heads"], case["kv_heads"]
    out = torch.empty_like(t["q"])
    if case["op"] == "append":
        QA.check(L.qwen_hip_paged_append(*t["by"], out.data_ptr(), ptr("q"), ptr("k"), ptr("v"), t["act"], H * HD,
                                         KH * HD, H, ptr("q_norm"), ptr("k_norm"), EPS, ptr("cos"), ptr("sin"),
                                         t["cos"].shape[0], s), "paged_append")
        return [out, t["k_pages"], t["v_pages"]]
    call = L.qwen_hip_paged_attention_decode if case["op"] == "decode" else L.qwen_hip_paged_attention_prefill
    QA.check(call(*t["by"], out.data_ptr(), ptr("q"), t["act"], H, SCALE, ptr("ws"), t["ws"].numel(), s), case["op"])
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        # a comparison, an exponential and a sum for each entry
        return {"bytes": 4.0 * case["rows"] * case["vocab"] + 24 * case["rows"], "flops": 4.0 * case["rows"] * case["vocab"]}
    new, lens = _shape(case)
    KH, a, c = case["kv_heads"], SIZE[case["act"]], SIZE[case["cache"]]
    H, rows, n = case["group"] * KH, sum(new), case["seqs"]
    page_ids = 4.0 * sum(-(-l // case["page"]) for l in lens)
    if case["op"] == "append":
        b = rows * HD * (a * (2 * H + 2 * KH) + c * 2 * KH) + 2 * 4 * HD * (max(lens) - min(l - m for l, m in zip(lens, new)))
        return {"bytes": float(b + 8 * n + 4 * rows), "flops": 8.0 * rows * (H + KH) * HD}
    pairs = sum(m * (l - m) + m * (m + 1) / 2 for m, l in zip(new, lens))
    b = 2 * a * rows * H * HD + 2 * c * KH * HD * sum(lens) + page_ids + 8 * n
    return {"bytes": float(b), "flops": 4.0 * HD * H * pairs}


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def exact(case, seed):
    t = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(t)
    KH, G, ps = case["kv_heads"], case["group"], case["page"]
    new, lens = _shape(case)
    if case["op"] == "append":
        return _exact_append(t, new, lens)
    out, at = [], 0
    for s, (m, l) in enumerate(zip(new, lens)):
        ids = t["table"][s, : -(-l // ps)].long()
        k, v = (x[ids].double().transpose(0, 1).reshape(KH, -1, HD)[:, :l] for x in (t["k_pages"], t["v_pages"]))
        q = t["q"][at:at + m].double().view(m, KH, G, HD)
        mask = torch.ones(m, l, dtype=torch.bool, device="cuda").tril(l - m)
        heads = []
        for h in range(KH):
            for g in range(G):
                s_ = (q[:, h, g] @ k[h].t()) / math.sqrt(HD)
                heads.append(torch.softmax(s_.masked_fill(~mask, -math.inf), -1) @ v[h])
        out.append(torch.cat(heads, 1))
        at += m
    return torch.cat(out)


def _exact_append(t, new, lens):
    case = t["case"]
    KH, ps = case["kv_heads"], case["page"]
    out, at, kp, vp = [], 0, t["k_pages"].double(), t["v_pages"].double()

    def turned(x, w, p0):
        m = x.shape[0]
        x = x.double().view(m, -1, 2, HD // 2)
        x = x / torch.sqrt((x * x).sum((2, 3), keepdim=True) / HD + EPS) * w.double().view(2, HD // 2)
        c, s = (t[n][p0:p0 + m, :HD // 2].double()[:, None] for n in ("cos", "sin"))
        return torch.stack([x[:, :, 0] * c - x[:, :, 1] * s, x[:, :, 1] * c + x[:, :, 0] * s], 2).view(m, -1, HD)

    for s, (m, l) in enumerate(zip(new, lens)):
        rows = slice(at, at + m)
        out.append(turned(t["q"][rows], t["q_norm"], l - m).reshape(m, -1))
        p = torch.arange(l - m, l, device="cuda")
        # the sequence's pages as rows of one slot each, through the table
        where = t["table"][s].long()[torch.div(p, ps, rounding_mode="floor")] * ps + p % ps
        for pages, x in ((kp, turned(t["k"][rows], t["k_norm"], l - m)), (vp, t["v"][rows].double().view(m, KH, HD))):
            flat = pages.transpose(1, 2).reshape(-1, KH, HD)
            flat[where] = x
            pages.copy_(flat.view(-1, ps, KH, HD).transpose(1, 2))
        at += m
    return [torch.cat(out), kp, vp]


def _exact_sample(t):
    got = []
    for r in range(t["case"]["rows"]):
        x, T, u = t["logits"][r].cpu().numpy().astype(np.float64), float(t["temperature"][r]), float(t["u"][r])
        k, p, least = int(t["top_k"][r]), float(t["top_p"][r]), float(t["min_p"][r])
        order = np.argsort(-x, kind="stable")
        if k > 0:
            order = order[:k]
        w = np.exp((x[order] - x[order[0]]) / T)
        if p < 1:
            n = int(np.sum(np.concatenate([[0.0], np.cumsum(w)[:-1]]) < p * w.sum()))
            order, w = order[:n], w[:n]
        order, w = order[w >= least], w[w >= least]
        by_index = np.argsort(order)
        order, cdf = order[by_index], np.cumsum(w[by_index])
        got.append(int(order[min(len(order) - 1, np.searchsorted(cdf, u * cdf[-1], side="right"))]))
    return np.array(got, np.int32)

"""The serving operators over a paged key-value cache, as cases to measure: attention of one new token per sequence
(optionally with a sliding window and first tokens that stay visible), appending rotated keys and values to the pages,
and managing the pages (fork, extend, free, compact).

`own` false: elementary torch operations in fp32; true: the calls of smlm_b200.paged.

Lengths of a batch follow from the case ("spread" over 0..len); a seed permutes them and makes the values.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _paged():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-memory-lm_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from smlm_b200 import paged
    return paged


# ------------------------------------------------------------------------------------------------- cases
def _attention(name, batch, hq, hkv, d, page, length, spread="same", dtype="bf16", window=0, sinks=0, order="hnd"):
    return {"name": name, "op": "attention", "batch": batch, "hq": hq, "hkv": hkv, "d": d, "page": page,
            "len": length, "spread": spread, "dtype": dtype, "window": window, "sinks": sinks, "order": order}


def _append(name, batch, tokens, hq, hkv, d, page, length, spread="same", dtype="bf16"):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d,
            "page": page, "len": length, "spread": spread, "dtype": dtype}


def _pages(name, op, rows, children, hkv, d, page, length, layers, dtype="bf16", new=1):
    return {"name": name, "op": op, "rows": rows, "children": children, "hkv": hkv, "d": d, "page": page,
            "len": length, "layers": layers, "dtype": dtype, "new": new}


def listed():
    return [
        # one sequence of the model's own shape (6 heads of 64) at the end of a 2048-token prompt + 256 new tokens
        _attention("decode-1", 1, 6, 6, 64, 16, 2304),
        # the same model serving 64 sequences, in the middle of their 256 new tokens
        _attention("decode-64", 64, 6, 6, 64, 16, 2175),
        # a server's mixed batch: shared key heads, sequences from nothing cached to 8k tokens
        _attention("decode-ragged", 96, 32, 8, 128, 32, 8191, spread="log"),
        # one very long document
        _attention("decode-long", 1, 32, 8, 128, 64, 131071, dtype="f16"),
        # streams that keep their first 4 tokens and the last 1024
        _attention("decode-window", 64, 16, 2, 128, 16, 20011, spread="even", window=1024, sinks=4),
        # fp32 decoding (no autocast) of uneven sequences, heads next to each other in a page
        _attention("decode-f32", 8, 6, 6, 64, 16, 1023, spread="even", dtype="f32", order="nhd"),
        # one decoding step of 64 sequences: this layer's new keys and values
        _append("append-step", 64, 1, 6, 6, 64, 16, 2175, spread="even"),
        # 16 prompts of 2048 tokens
        _append("append-prompts", 16, 2048, 6, 6, 64, 16, 2048),
        # a chunk of 777 tokens after cached ones, fp32, shared key heads
        _append("append-chunk-f32", 3, 777, 32, 8, 128, 32, 2001, spread="even", dtype="f32"),
        # eight samples of one prompt: the last samples dropped, forked again, one token added
        _pages("fork-8", "fork", 1, 8, 6, 64, 16, 1001, 6),
        # 16 prompts with 16 samples each
        _pages("fork-256", "fork", 16, 256, 6, 64, 64, 2031, 6),
        # a cache of which every second sequence has ended, compacted
        _pages("compact-half", "compact", 90, 0, 6, 64, 16, 1024, 6),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _avoid(case):
    """Keeps one much-used benchmark size out of the draws."""
    sizes = [v for v in case.values() if isinstance(v, int)]
    if "hq" in case:
        sizes += [(case["hq"] + 2 * case["hkv"]) * case["d"], case["hq"] * case["d"]]
    return 3072 in sizes


def draw(rng):
    while True:
        kind = rng.choice(["attention", "attention", "append", "pages"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        hq, hkv = rng.choice([(6, 6), (6, 6), (8, 1), (12, 4), (16, 2), (24, 24), (32, 8), (7, 7), (20, 10)])
        d = rng.choice([16, 32, 64, 64, 64, 80, 96, 128, 128, 256])
        page = rng.choice([8, 16, 16, 32, 64, 128])
        if kind == "attention":
            batch, length = _log(rng, 1, 128), _log(rng, 1, 131072)
            window = rng.choice([0, 0, _log(rng, 8, 8192)])
            case = _attention("", batch, hq, hkv, d, page, length, rng.choice(["same", "even", "log"]), dtype, window,
                              rng.choice([0, 1, 4, 33]) if window else 0, rng.choice(["hnd", "hnd", "nhd"]))
            held = sum(_lengths(case)) * hkv * d * 2 * BYTES[dtype]
            if held > 540e6 or batch * length * hkv * d > 600e6:
                continue
        elif kind == "append":
            batch, tokens = _log(rng, 1, 128), _log(rng, 1, 4096)
            length = tokens + _log(rng, 1, 4096)
            case = _append("", batch, tokens, hq, hkv, d, page, length, rng.choice(["same", "even"]), dtype)
            if batch * length * (hq + 2 * hkv) * d * BYTES[dtype] > 300e6:
                continue
        else:
            op = rng.choice(["fork", "compact"])
            layers, length, rows = rng.choice([1, 6, 12]), _log(rng, 16, 4096), _log(rng, 1, 64)
            case = _pages("", op, rows if op == "fork" else rows + 2, _log(rng, 1, 16) * rows if op == "fork" else 0,
                          hkv, d, page, length, layers, dtype, rng.choice([1, 1, 17]))
            if rows * length * hkv * d * 2 * BYTES[dtype] * layers > 600e6:
                continue
            if case["children"] * page * hkv * d * 2 * BYTES[dtype] * layers > 300e6:
                continue
        if _avoid(case):
            continue
        del case["name"]
        return case


def _lengths(case):
    """The batch's lengths, in increasing order (from the case alone)."""
    n, top = case["batch"], case["len"]
    if case["spread"] == "same" or n == 1:
        return [top] * n
    if case["spread"] == "even":
        return [max(1, top * (i + 1) // n) for i in range(n)]
    return [0] + [int(round(top ** (i / (n - 1)))) for i in range(1, n)]


def _visible(case, n):
    w = case["window"]
    if not w or n <= w:
        return n
    return w + min(case["sinks"], n - w)


def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] == "attention":
        seen = sum(_visible(case, n) for n in _lengths(case))
        qo = 2 * case["batch"] * case["hq"] * case["d"] * es
        return {"bytes": seen * case["hkv"] * case["d"] * 2 * es + qo + 4 * (seen // case["page"] + case["batch"]),
                "flops": 4 * seen * case["hq"] * case["d"]}
    if case["op"] == "append":
        tokens = sum(min(n, case["tokens"]) for n in _lengths(case))
        wide = (case["hq"] + 2 * case["hkv"]) * case["d"]
        return {"bytes": 2 * tokens * wide * es + tokens * case["d"] * 4,
                "flops": 3 * tokens * (case["hq"] + case["hkv"]) * case["d"]}
    token = 2 * case["layers"] * case["hkv"] * case["d"] * es
    if case["op"] == "fork":
        lens = _fork_lengths(case)
        moved = sum(lens[i % case["rows"]] % case["page"] for i in range(case["children"]))
        entries = sum(lens[i % case["rows"]] // case["page"] for i in range(case["children"]))
        return {"bytes": 2 * moved * token + 12 * entries, "flops": 0}
    pages, live, moves = _compact_counts(case)
    return {"bytes": 2 * moves * case["page"] * token + 8 * live + 4 * pages, "flops": 0}


# ----------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rope(d, n):
    freq = 1.0 / 10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d)
    angle = torch.arange(n, dtype=torch.float32)[:, None] * freq[None]
    return angle.cos().cuda(), angle.sin().cuda()


def _table(blocks, extra, r):
    """Pages of a pool that has been in use for a while: every sequence's pages lie anywhere in it."""
    pages = sum(blocks) + extra
    order = r.permutation(pages)
    table = np.full((len(blocks), max(1, max(blocks))), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def _cdiv(a, b):
    return -(-a // b)


def _fork_lengths(case):
    r = random.Random(case["rows"] * 7919 + case["len"])
    return [max(1, case["len"] - r.randrange(0, max(1, min(case["len"], 4 * case["page"])))) for _ in range(case["rows"])]


def _compact_layout(case):
    """The pool of a compaction (from the case alone): sequences of `len` tokens, every second one ended."""
    r = np.random.RandomState(case["rows"] * 31 + case["len"])
    blocks = [_cdiv(case["len"], case["page"])] * case["rows"]
    table, pages = _table(blocks, max(2, sum(blocks) // 8), r)
    table[1::2] = -1
    return table, pages


def _compact_counts(case):
    table, pages = _compact_layout(case)
    live = int((table >= 0).sum())
    return pages, live, int((table >= live).sum())


def _prepare_tokens(case, seed):
    g, r = _gen(seed), np.random.RandomState(seed % (1 << 31))
    dtype = DTYPES[case["dtype"]]
    lens = [_lengths(case)[i] for i in r.permutation(case["batch"])]
    blocks = [_cdiv(n, case["page"]) for n in lens]
    table, pages = _table(blocks, max(1, sum(blocks) // 8), r)
    if case.get("order") == "nhd":       # a page holds token after token, each with all its heads
        pool = torch.randn(2, pages, case["page"], case["hkv"], case["d"], generator=g, device="cuda",
                           dtype=dtype).transpose(2, 3)
    else:                                # a page holds head after head
        pool = torch.randn(2, pages, case["hkv"], case["page"], case["d"], generator=g, device="cuda", dtype=dtype)
    return {"case": case, "g": g, "k": pool[0], "v": pool[1], "table": torch.from_numpy(table).cuda(),
            "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    if case["op"] == "attention":
        s = _prepare_tokens(case, seed)
        s["q"] = torch.randn(case["batch"], case["hq"], case["d"], generator=s["g"], device="cuda",
                             dtype=DTYPES[case["dtype"]])
        return s
    if case["op"] == "append":
        s = _prepare_tokens(case, seed)
        wide = (case["hq"] + 2 * case["hkv"]) * case["d"]
        s["qkv"] = torch.randn(case["batch"], case["tokens"], wide, generator=s["g"], device="cuda",
                               dtype=DTYPES[case["dtype"]])
        s["cos"], s["sin"] = _rope(case["d"], case["len"])
        return s
    g, r = _gen(seed), np.random.RandomState(seed % (1 << 31))
    page, dtype = case["page"], DTYPES[case["dtype"]]
    if case["op"] == "fork":
        lens = _fork_lengths(case)
        shared = [_cdiv(n, page) for n in lens]
        # room for every child's own last page and its new tokens
        table, pages = _table(shared, case["children"] * (2 + _cdiv(case["new"], page)) + 3, r)
        width = max(_cdiv(n + case["new"], page) for n in lens)
        full = np.full((case["rows"] + case["children"], width), -1, dtype=np.int32)
        full[:case["rows"], :table.shape[1]] = table
        lens = lens + [0] * case["children"]
        table = full
    else:
        table, pages = _compact_layout(case)
        lens = [case["len"] if table[i, 0] >= 0 else 0 for i in range(case["rows"])]
    refcount = np.zeros(pages, dtype=np.int32)
    refcount[table[table >= 0]] = 1
    s = {"case": case, "table": torch.from_numpy(table).cuda(), "refcount": torch.from_numpy(refcount).cuda(),
         "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "pool": torch.randn(case["layers"], 2, pages, case["hkv"], page, case["d"], generator=g, device="cuda",
                             dtype=dtype)}
    if case["op"] == "fork":
        ids = torch.arange(case["children"], dtype=torch.int32, device="cuda")
        s["parents"], s["children"] = ids % case["rows"], ids + case["rows"]
    else:                                # what the compaction changes, to begin each pass with
        s["table0"], s["refcount0"] = s["table"].clone(), s["refcount"].clone()
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_attention(q, k_pages, v_pages, table, lengths, window, sinks):
    B, hq, d = q.shape
    hkv, page = k_pages.shape[1], k_pages.shape[2]
    pages = table.clamp(min=0).long()
    k = k_pages[pages].float().transpose(1, 2).reshape(B, hkv, -1, d)
    v = v_pages[pages].float().transpose(1, 2).reshape(B, hkv, -1, d)
    j = torch.arange(table.shape[1] * page, device=q.device)[None]
    n = lengths[:, None]
    seen = (j < n) & (table >= 0).repeat_interleave(page, dim=1)
    if window:
        seen &= (j >= n - window) | (j < sinks)
    s = torch.matmul(q.float().view(B, hkv, hq // hkv, d), k.transpose(2, 3)) * d ** -0.5
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return out.view(B, hq, d).to(q.dtype)


def _plain_append(qkv, k_pages, v_pages, table, lengths, cos, sin):
    B, T, wide = qkv.shape
    hkv, page, d = k_pages.shape[1:]
    hq = wide // d - 2 * hkv
    at = lengths[:, None].long() - T + torch.arange(T, device=qkv.device)
    held = at >= 0
    at = at.clamp(min=0)
    x = qkv.view(B, T, hq + 2 * hkv, d).float()
    a, b = x[:, :, :hq + hkv].chunk(2, dim=-1)
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    pages, slots = table.long().gather(1, at // page)[held], (at % page)[held]
    k_pages[pages, :, slots] = turned[:, :, hq:].to(k_pages.dtype)[held]
    v_pages[pages, :, slots] = x[:, :, hq + hkv:].to(v_pages.dtype)[held]
    return (turned[:, :, :hq] * held[:, :, None, None]).to(qkv.dtype)


def _plain_free(table, lengths, refcount, rows):
    rows = rows.long()
    old = table[rows]
    old = old[old >= 0].long()
    refcount.index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    table[rows] = -1
    lengths[rows] = 0


def _plain_fork(pool, table, lengths, refcount, parents, children):
    page = pool.shape[4]
    one = torch.ones_like(refcount)
    p, c = parents.long(), children.long()
    rows, n = table[p], lengths[p].long()
    full, part = n // page, n % page
    shared = (torch.arange(table.shape[1], device=table.device)[None] < full[:, None]) & (rows >= 0)
    refcount.index_add_(0, rows[shared].long(), one[:1].expand(int(shared.sum())))
    src = rows.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    has = (part > 0) & (src >= 0)
    src, part = src[has], part[has]
    refcount.index_add_(0, src, one[:1].expand(len(src)))             # still needed while pages are given out
    old = table[c]
    old = old[old >= 0].long()
    refcount.index_add_(0, old, -one[:1].expand(len(old)))
    dst = torch.nonzero(refcount == 0)[:len(src), 0]
    refcount.index_add_(0, src, -one[:1].expand(len(src)))
    refcount[dst] = 1
    rows = torch.where(shared, rows, -1)
    rows[has.nonzero()[:, 0], full[has]] = dst.int()
    table[c] = rows
    lengths[c] = n.int()
    keep = torch.arange(page, device=table.device)[None] < part[:, None]
    pool[:, :, dst] = torch.where(keep[None, None, :, None, :, None], pool[:, :, src], pool[:, :, dst])


def _plain_extend(table, lengths, refcount, rows, new, page):
    rows = rows.long()
    n = lengths[rows]
    j = torch.arange(table.shape[1], device=table.device)[None]
    grow = (j >= ((n + page - 1) // page)[:, None]) & (j < ((n + new + page - 1) // page)[:, None])
    dst = torch.nonzero(refcount == 0)[:int(grow.sum()), 0]
    mine = table[rows]
    mine[grow] = dst.int()
    table[rows] = mine
    refcount[dst] = 1
    lengths[rows] = n + new


def _plain_compact(pool, table, refcount):
    live = refcount > 0
    n = int(live.sum())
    low, high = torch.nonzero(~live[:n])[:, 0], torch.nonzero(live[n:])[:, 0] + n
    pool[:, :, low] = pool[:, :, high]
    to = torch.arange(len(refcount), dtype=torch.int32, device=table.device)
    to[high] = low.int()
    refcount[low] = refcount[high]
    refcount[high] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))


def run(s):
    c = s["case"]
    op = _paged() if own else None
    if c["op"] == "attention":
        if own:
            return op.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=c["window"],
                                      sinks=c["sinks"])
        return _plain_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], c["window"], c["sinks"])
    if c["op"] == "append":
        append = op.paged_append if own else _plain_append
        q = append(s["qkv"], s["k"], s["v"], s["table"], s["lengths"], s["cos"], s["sin"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["op"] == "fork":
        if own:
            op.pages_free(s["table"], s["lengths"], s["refcount"], s["children"])
            op.pages_fork(s["pool"], s["table"], s["lengths"], s["refcount"], s["parents"], s["children"])
            op.pages_extend(s["table"], s["lengths"], s["refcount"], s["children"], c["new"], c["page"])
        else:
            _plain_free(s["table"], s["lengths"], s["refcount"], s["children"])
            _plain_fork(s["pool"], s["table"], s["lengths"], s["refcount"], s["parents"], s["children"])
            _plain_extend(s["table"], s["lengths"], s["refcount"], s["children"], c["new"], c["page"])
    else:
        s["table"].copy_(s["table0"])
        s["refcount"].copy_(s["refcount0"])
        compact = op.pages_compact if own else _plain_compact
        compact(s["pool"], s["table"], s["refcount"])
    return {"pool": s["pool"], "table": s["table"], "lengths": s["lengths"], "refcount": s["refcount"]}


# -------------------------------------------------------------------------------------------- 64 bits
def _exact_attention(s):
    c = s["case"]
    lens, table = s["lengths"].tolist(), s["table"].long()
    group = c["hq"] // c["hkv"]
    out = torch.zeros(c["batch"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        if c["window"]:
            at = at[(at >= n - c["window"]) | (at < c["sinks"])]
        if not len(at):
            continue
        pages, slots = table[b, at // c["page"]], at % c["page"]
        for h in range(c["hkv"]):
            k, v = s["k"][pages, h, slots].double(), s["v"][pages, h, slots].double()
            q = s["q"][b, h * group:(h + 1) * group].double()
            w = torch.softmax(q @ k.T / math.sqrt(c["d"]), dim=-1)
            out[b, h * group:(h + 1) * group] = w @ v
    return out


def _exact_append(s):
    c = s["case"]
    half, nq = c["d"] // 2, c["hq"] + c["hkv"]
    k, v = s["k"].double(), s["v"].double()
    q = torch.zeros(c["batch"], c["tokens"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        skip = max(0, c["tokens"] - n)
        at = torch.arange(n - c["tokens"] + skip, n, device="cuda")
        x = s["qkv"][b, skip:].double().reshape(len(at), c["hq"] + 2 * c["hkv"], c["d"])
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.atan2(s["sin"][at].double(), s["cos"][at].double()))
        size = torch.hypot(s["sin"][at].double(), s["cos"][at].double())
        z = torch.complex(x[:, :nq, :half], x[:, :nq, half:]) * (turn * size)[:, None]
        x = torch.cat((torch.cat((z.real, z.imag), dim=-1), x[:, nq:]), dim=1)
        q[b, skip:] = x[:, :c["hq"]]
        pages, slots = s["table"][b].long()[at // c["page"]], at % c["page"]
        k[pages, :, slots] = x[:, c["hq"]:nq]
        v[pages, :, slots] = x[:, nq:]
    return {"q": q, "k": k, "v": v}


def _exact_pages(s):
    """The pool of a fork or a compaction, page by page as a reader of the tables sees it."""
    c, page = s["case"], s["case"]["page"]
    pool, count = s["pool"].double(), s["refcount"].tolist()
    table, lens = s["table"].tolist(), s["lengths"].tolist()
    if c["op"] == "fork":
        free = [i for i, n in enumerate(count) if n == 0]
        at = 0
        for parent in s["parents"].tolist():
            part = lens[parent] % page
            if part:
                pool[:, :, free[at], :, :part] = pool[:, :, table[parent][lens[parent] // page], :, :part]
                at += 1
    else:
        n = sum(x > 0 for x in count)
        low = [i for i in range(n) if count[i] == 0]
        high = [i for i in range(n, len(count)) if count[i] > 0]
        for a, b in zip(low, high):
            pool[:, :, a] = pool[:, :, b]
    return {"pool": pool, "table": None, "lengths": None, "refcount": None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append}.get(case["op"], _exact_pages)(s)

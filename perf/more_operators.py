"""Operators of a serving step as cases that can be timed and compared, plain forms beside the library's calls: a paged KV cache in
4 bits and its attention, the step's block tables and slot map from the requests' lengths, and the norms on both sides of a block.

A case is one of

* ``append``  new tokens' K and V written into 4-bit pages (with ``rope`` rotated on the way, the queries too) and read back;
* ``attend``  attention of the new tokens of every sequence (one, a few, a chunk, a whole prompt) over a cache in 4 bits;
* ``tables``  a step planned on the device (rows, pages from the free list, lengths, a slot for every row) and taken back, as after
              drafts that were rejected: lengths, tables and the free list are then what they were;
* ``norm``    residual_out = residual + scale * gate * norm(block), out = norm(residual_out).

A batch has ``seqs`` sequences.  ``chunks`` of them bring about ``new`` tokens each, the others one token; their cached lengths lie
between ``kv_min`` and ``kv_max`` (new tokens included) and are the same for every seed, so that the work of a case is known.
Pages are handed out in random order, as after some hours of serving.

A cached element is zero + scale * u, u in 0 .. 15, with one pair (scale, zero) in bf16 for each position and kv head.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ROPE_LEN = 16384
EPS = 1e-5


def _batch(kind, name=None, **kw):
    c = dict(kind=kind, seqs=1, chunks=0, new=1, kv_min=1, kv_max=1, heads=32, kv_heads=32, hd=128, page=16, io="bf16", window=0, sinks=0, rope=False, layout="NHD")
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def _norm(name=None, **kw):
    c = dict(kind="norm", rows=1, dim=4096, block="bf16", residual="f32", io="bf16", post=True, gate="none", scale=1.0)
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # A decode step of a small batch on the 7B shape: what the projections give (f32) is rotated and written; latency counts.
        _batch("append", "append4-step-7b", seqs=16, kv_min=40, kv_max=2000, io="f32", rope=True),
        # The chunks of several long prompts at once.
        _batch("append", "append4-chunks-13b", seqs=6, chunks=6, new=1500, kv_min=1500, kv_max=6000, heads=40, kv_heads=40, page=32),
        # One user, one token: the smallest call of serving.
        _batch("attend", "attend4-one-7b", kv_min=517, kv_max=517, io="f16"),
        # A full serving batch, very ragged, grouped query heads.
        _batch("attend", "attend4-step-70b", seqs=64, kv_min=1, kv_max=8192, heads=64, kv_heads=8),
        # Long streams with a bounded window and a few sinks.
        _batch("attend", "attend4-stream-13b-window", seqs=8, kv_min=20000, kv_max=60000, heads=40, kv_heads=40, page=32, window=4096, sinks=4),
        # Serving with chunked prompts: two chunks among single tokens.
        _batch("attend", "attend4-mixed-13b", seqs=26, chunks=2, new=389, kv_min=30, kv_max=2500, heads=40, kv_heads=40, layout="HND"),
        # The last chunk of a long document.
        _batch("attend", "attend4-chunk-70b", chunks=1, new=512, kv_min=15000, kv_max=15000, heads=64, kv_heads=8, page=64),
        # A decode step's tables: one token for each of a full batch.
        _batch("tables", "tables-step", seqs=64, kv_min=1, kv_max=8192),
        # Hundreds of requests, dozens of long prompts among them.
        _batch("tables", "tables-prompts", seqs=500, chunks=24, new=2000, kv_min=1, kv_max=4000),
        # Between two blocks of a decode step.
        _norm("norm-step-7b", rows=16, dim=4096),
        # Post-norm with a gate for each channel, after a chunk of a prompt: an odd number of rows.
        _norm("norm-chunk-13b-gate", rows=389, dim=5120, residual="bf16", gate="channel", scale=0.5),
        # A long prompt on the 70B shape, residual stream in f32.
        _norm("norm-prompt-70b", rows=8191, dim=8192, post=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    most = _cost(listed()[6])
    while True:
        kind = rng.choice(["append", "attend", "attend", "attend", "attend", "tables", "norm", "norm"])
        if kind == "norm":
            c = _norm(rows=_log(rng, 1, 8191), dim=rng.choice([_log(rng, 64, 16384), 8 * _log(rng, 8, 2048), 4096, 5120, 8192]), block=rng.choice(["bf16", "f16", "f32"]),
                      residual=rng.choice(["f32", "bf16", "f16"]), io=rng.choice(["bf16", "f16"]), post=rng.random() < 0.6,
                      gate=rng.choice(["none", "channel", "element"]), scale=rng.choice([1.0, 0.5, 0.22]))
            if c["rows"] * c["dim"] <= 8191 * 8192:
                return c
            continue
        kv_heads, group = rng.choice([(32, 1), (40, 1), (8, 8), (8, 4), (4, 2), (2, 8), (1, 16), (4, 3), (16, 1)])
        c = _batch(kind, heads=kv_heads * group, kv_heads=kv_heads, hd=rng.choice([128, 128, 128, 64]), page=rng.choice([16, 32, 64, 128]),
                   io=rng.choice(["bf16", "bf16", "f16"]), layout=rng.choice(["NHD", "HND"]))
        c["seqs"] = _log(rng, 1, 2000 if kind == "tables" else 128)
        c["kv_max"] = _log(rng, 2, 65536 if c["seqs"] < 8 else 8192)
        c["kv_min"] = rng.randint(1, c["kv_max"])
        if rng.random() < 0.6:
            c["chunks"] = rng.randint(1, max(1, min(c["seqs"], 8)))
            c["new"] = _log(rng, 2, 8191)
            c["kv_max"] = max(c["kv_max"], c["new"] + 1)
        if kind == "append":
            c["rope"] = rng.random() < 0.5 and c["kv_max"] <= ROPE_LEN
            if c["rope"]:
                c["io"] = rng.choice(["f32", c["io"]])
        if kind == "attend" and rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 16, 8192), rng.choice([0, 1, 4, 17, 64])
        if _cost(c) <= most and _plain_bytes(c) <= 25e9:
            return c


def _lengths(case):
    """(rows, cached tokens) of every sequence: spread over the range by the golden ratio, the same for every seed."""
    u = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(case["seqs"])]
    rows = [1 + int((0.75 + 0.25 * x) * (case["new"] - 1)) if i < case["chunks"] else 1 for i, x in enumerate(u)]
    if case["chunks"] == 1:
        rows[0] = case["new"]
    kv = [int(round(case["kv_min"] + x * (case["kv_max"] - case["kv_min"]))) for x in u]
    if case["seqs"] == 1:
        kv[0] = case["kv_max"]
    return rows, [max(a, b) for a, b in zip(kv, rows)]


def _pairs(case):
    """Visible (row, key) pairs of the batch, and the distinct keys that its rows see."""
    rows, kv = _lengths(case)
    w, sinks = case["window"], case["sinks"]

    def upto(n):  # sum over positions p < n of the keys that p sees
        if w == 0 or n <= w:
            return n * (n + 1) // 2
        full = w * (w + 1) // 2 + (n - w) * w
        m = n - w  # positions w .. n - 1 see min(sinks, p - w + 1) keys in front of their window
        return full + (m * (m + 1) // 2 if m <= sinks else sinks * (sinks + 1) // 2 + (m - sinks) * sinks)

    pairs = sum(upto(k) - upto(k - r) for r, k in zip(rows, kv))
    keys = sum(k if w == 0 else k - max(0, k - r - w + 1) + min(sinks, max(0, k - r - w + 1)) for r, k in zip(rows, kv))
    return pairs, keys


def _plain_bytes(case):
    rows, kv = _lengths(case)
    if case["kind"] == "tables":
        return 40 * (case["seqs"] * (-(-max(kv) // case["page"]) + 1) + sum(rows))
    caches = 2 * case["seqs"] * max(kv) * case["kv_heads"] * case["hd"] * 4
    return caches + (12 * case["seqs"] * max(rows) * case["heads"] * max(kv) if case["kind"] == "attend" else 0)


def _cost(case):
    """About what the plain form takes, in bytes moved."""
    return 4 * _plain_bytes(case) + work(case)["bytes"] + (4 * case["hd"] * case["seqs"] * max(_lengths(case)[0]) * case["heads"] * max(_lengths(case)[1]) / 10 if case["kind"] == "attend" else 0)


def work(case):
    if case["kind"] == "norm":
        n = case["rows"] * case["dim"]
        gate = {"none": 0, "channel": 2 * case["dim"], "element": 2 * n}[case["gate"]]
        weights = 4 * case["dim"] * (2 if case["post"] else 1)
        return {"bytes": n * (SIZE[case["block"]] + 2 * SIZE[case["residual"]] + SIZE[case["io"]]) + gate + weights, "flops": 0}
    rows, kv = _lengths(case)
    n, row = sum(rows), case["kv_heads"] * case["hd"]
    if case["kind"] == "tables":
        # the plan: a sequence's length and rows in, its length and first row out; a page from the free list into the table for each new one; a
        # slot and a position for each row.  And back: lengths in and out, the pages.
        pages = sum(-(-b // case["page"]) + -((a - b) // case["page"]) for a, b in zip(rows, kv))
        return {"bytes": case["seqs"] * (16 + 12) + 8 * pages + 12 * n + 12 * pages, "flops": 0}
    held = 2 * (row // 2 + 4 * case["kv_heads"])  # K and V of a cached token, with a pair of bf16 for each kv head
    q_row = case["heads"] * case["hd"]
    if case["kind"] == "attend":
        pairs, keys = _pairs(case)
        return {"bytes": keys * held + 2 * n * q_row * SIZE[case["io"]], "flops": 4.0 * case["hd"] * case["heads"] * pairs}
    queries = n * q_row * (SIZE[case["io"]] + 2) if case["rope"] else 0
    return {"bytes": n * (2 * held + 2 * row * SIZE[case["io"]] + 2 * row * 2) + queries, "flops": 0}


def _floats(gen, shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"append": _prepare_cache, "attend": _prepare_cache, "tables": _prepare_tables, "norm": _prepare_norm}[case["kind"]](case, gen)


def _page_table(case, kv, extra, gen):
    """Pages in random order: (table, -1 where there is none, number of pages, the free ones in random order)."""
    page = case["page"]
    width = -(-max(kv) // page) + 1
    used = [-(-x // page) for x in kv]
    n_pages = sum(used) + extra
    order = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)
    seq = torch.repeat_interleave(torch.arange(len(used)), torch.tensor(used))
    first = torch.tensor([0] + used).cumsum(0)
    col = torch.arange(sum(used)) - first[seq]
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    table[seq.cuda(), col.cuda()] = order[: sum(used)]
    return table, n_pages, order[sum(used):].clone()


def _prepare_tables(case, gen):
    rows, kv = _lengths(case)
    before = [k - r for r, k in zip(rows, kv)]
    extra = sum(-(-k // case["page"]) - -(-b // case["page"]) for k, b in zip(kv, before)) + 8
    table, n_pages, free = _page_table(dict(case, kv_max=max(kv)), before, extra, gen)
    width = -(-max(kv) // case["page"]) + 1
    room = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    room[:, : min(width, table.shape[1])] = table[:, :width]
    stack = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    stack[: len(free)] = free
    n = sum(rows) + 5  # a little more room than rows, as a captured step has
    s = {"case": case, "table": room, "kv_len": _ints(before), "keep": _ints(before), "free": stack, "free_count": _ints([len(free)]), "new_rows": _ints(rows),
         "row_start": torch.zeros(len(kv) + 1, dtype=torch.int32, device="cuda"), "slots": torch.zeros(n, dtype=torch.int64, device="cuda"),
         "positions": torch.zeros(n, dtype=torch.int32, device="cuda"), "n": n, "max_rows": max(rows)}
    if own:
        s["tables"] = _package().KvTables(s["table"], s["kv_len"], s["free"], s["free_count"], case["page"])
    return s


def _prepare_norm(case, gen):
    n, dim = case["rows"], case["dim"]
    s = {"case": case, "block": _floats(gen, (n, dim), TYPES[case["block"]]), "residual": _floats(gen, (n, dim), TYPES[case["residual"]]), "post": None, "gate": None}
    s["residual"] *= 3
    s["pre"] = 1 + 0.2 * _floats(gen, (dim,), torch.float32)
    if case["post"]:
        s["post"] = 1 + 0.2 * _floats(gen, (dim,), torch.float32)
    if case["gate"] != "none":
        s["gate"] = _floats(gen, (dim,) if case["gate"] == "channel" else (n, dim), torch.bfloat16)
    s["residual_out"], s["out"] = torch.empty_like(s["residual"]), torch.empty((n, dim), dtype=TYPES[case["io"]], device="cuda")
    if own:
        s["package"] = _package()
    return s


def _prepare_cache(case, gen):
    rows, kv = _lengths(case)
    n, page, kvh, hd = sum(rows), case["page"], case["kv_heads"], case["hd"]
    table, n_pages, _ = _page_table(case, kv, 8, gen)
    row_start = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    row_seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    s = {
        "case": case, "table": table, "row_start": row_start.cuda(), "kv_len": _ints(kv),
        "n": n, "max_rows": max(rows), "max_kv": max(kv), "scale": 1.0 / math.sqrt(hd),
        # where each row is: its sequence, its place in it and its position
        "row_seq": row_seq.cuda(), "row_at": (torch.arange(n) - row_start[row_seq]).cuda(),
        "row_pos": (torch.arange(n) - row_start[row_seq] + torch.tensor(kv)[row_seq] - torch.tensor(rows)[row_seq]).cuda(),
    }
    io = TYPES[case["io"]]
    shape = (n_pages, page, kvh, hd // 2) if case["layout"] == "NHD" else (n_pages, kvh, page, hd // 2)
    for x in "kv":
        s[x] = torch.empty(shape, dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
        step = torch.empty((n_pages, kvh, page, 2), device="cuda").uniform_(0.15, 0.35, generator=gen)
        step[..., 1] *= -30 * step[..., 0]  # the zero: half of the range below 0, more or less
        s[x + "_scale"] = step.to(torch.bfloat16)
    rounded = torch.bfloat16 if io == torch.float32 else io
    if case["kind"] == "append":
        # channels differ in size, as keys' do
        channel = torch.empty((kvh, hd), device="cuda").normal_(generator=gen).mul_(0.7).exp_()
        s["new_k"] = (_floats(gen, (n, kvh, hd), torch.float32) * channel).to(io)
        s["new_v"] = _floats(gen, (n, kvh, hd), io)
        if case["rope"]:
            s["q"], s["q_out"] = _floats(gen, (n, case["heads"], hd), io), torch.empty((n, case["heads"], hd), dtype=rounded, device="cuda")
            angle = torch.arange(ROPE_LEN).double()[:, None] * 10000.0 ** (-torch.arange(hd // 2).double() / (hd // 2))
            s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
        s["k_back"], s["v_back"] = (torch.empty((n, kvh, hd), dtype=rounded, device="cuda") for _ in "kv")
    else:
        s["q"], s["out"] = _floats(gen, (n, case["heads"], hd), io), torch.empty((n, case["heads"], hd), dtype=io, device="cuda")
    if own:  # the handles that a program keeps: the cache's pages, the step's batch (one for all layers), a workspace
        l2 = _package()
        s["pages"] = l2.KvPages(s["k"], s["v"], s["k_scale"], s["v_scale"], layout=case["layout"])
        s["batch"] = l2.KvBatch(s["table"], s["kv_len"], s["row_start"], s["n"], s["max_rows"])
        if case["kind"] == "attend":
            s["workspace"] = torch.empty(s["pages"].workspace_bytes(s["batch"], case["heads"]), dtype=torch.uint8, device="cuda")
    return s


def _package():
    path = os.path.join(os.getcwd(), "llama2.rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import llama2_rs
    return llama2_rs


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "tables": _own_tables, "norm": _own_norm}[kind](s)
    return {"append": _plain_append, "attend": _plain_attend, "tables": _plain_tables, "norm": _plain_norm}[kind](s)


# ---- the library's calls -------------------------------------------------------------------------------------------------

def _own_append(s):
    rope = (s["cos"], s["sin"]) if s["case"]["rope"] else None
    s["pages"].append(s["batch"], s["new_k"], s["new_v"], rope=rope, q=s.get("q"), q_out=s.get("q_out"))
    s["pages"].read(s["batch"], s["k_back"], s["v_back"])
    return {"k": s["k_back"], "v": s["v_back"], "q": s.get("q_out")}


def _own_attend(s):
    c = s["case"]
    s["pages"].attend(s["batch"], s["q"], s["out"], scale=s["scale"], window=c["window"], sinks=c["sinks"], workspace=s["workspace"])
    return s["out"]


def _own_tables(s):
    t = s["tables"]
    t.plan(s["new_rows"], s["row_start"], s["n"], s["max_rows"], slots=s["slots"], positions=s["positions"])
    t.release(s["keep"])
    return {k: s[k] for k in ("row_start", "slots", "positions", "kv_len", "table", "free", "free_count")}


def _own_norm(s):
    s["package"].block_norm(s["block"], s["residual"], s["out"], residual_out=s["residual_out"], post_weight=s["post"], pre_weight=s["pre"], gate=s["gate"],
                            scale=s["case"]["scale"], eps=EPS)
    return {"residual": s["residual_out"], "out": s["out"]}


# ---- plain forms: elementary operations in 32 bits, rounded once ----------------------------------------------------------

def _pool(s, name):
    """A view [page][token][kv head] of a pool, whatever its layout."""
    return s[name] if s["case"]["layout"] == "NHD" else s[name].transpose(1, 2)


def _slots(s):
    page = s["case"]["page"]
    return s["table"][s["row_seq"], s["row_pos"] // page].long(), s["row_pos"] % page


def _rotate(x, cos, sin):
    a, b = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_append(s):
    k, v, q = s["new_k"].float(), s["new_v"].float(), None
    if s["case"]["rope"]:
        cos, sin = s["cos"][s["row_pos"]][:, None], s["sin"][s["row_pos"]][:, None]
        k, q = _rotate(k, cos, sin), _rotate(s["q"].float(), cos, sin).to(s["q_out"].dtype)
    page, at = _slots(s)
    _quantise(s, "k", k, page, at)
    _quantise(s, "v", v, page, at)
    return {**{x: _values(s, x, page, at).to(s["k_back"].dtype) for x in "kv"}, "q": q}


def _quantise(s, name, x, page, at):
    """zero: the bf16 number at or below the least element; scale: the least bf16 number whose 15 steps reach the largest.  u goes by the product with
    the scale's reciprocal in 32 bits, which is taken in 64: elements of 16 bits often lie next to the middle of a step."""
    low = x.amin(-1, keepdim=True).view(torch.int32)
    zero = torch.where(low < 0, low + 0xffff, low).bitwise_and(-65536).view(torch.float32)
    span = x.amax(-1, keepdim=True) - zero
    scale = (span * (1.0 / 15.0)).view(torch.int32).bitwise_and(-65536)
    scale = torch.where(scale.view(torch.float32) * 15.0 < span, scale + 65536, scale).view(torch.float32)
    scale = torch.where(span < 2.0**-100, torch.zeros((), device="cuda"), scale)
    u = torch.round((x - zero).double() * scale.reciprocal().double())
    u = torch.where(scale > 0, u, torch.zeros((), dtype=torch.float64, device="cuda")).to(torch.uint8)
    _pool(s, name)[page, at] = u[..., 0::2] | (u[..., 1::2] << 4)
    s[name + "_scale"].transpose(1, 2)[page, at] = torch.cat((scale, zero), -1).to(torch.bfloat16)


def _values(s, name, page, at):
    x = _pool(s, name)[page, at]
    x = torch.stack((x & 15, x >> 4), -1).flatten(-2).float()
    pair = s[name + "_scale"].transpose(1, 2)[page, at].float()
    return pair[..., 1:] + pair[..., :1] * x


def _plain_attend(s):
    c = s["case"]
    kvh, hd, page, group = c["kv_heads"], c["hd"], c["page"], c["heads"] // c["kv_heads"]
    # every sequence's keys and values, padded to the longest: [sequence][kv head][position][hd]
    at = torch.arange(s["max_kv"], device="cuda")
    pages = s["table"][:, at // page].long().clamp_min(0)
    k, v = (_values(s, x, pages, at % page).transpose(1, 2) for x in "kv")
    # the rows, padded to the most: [sequence][kv head][row and query head of the group][hd]
    m = s["max_rows"]
    row = (s["row_start"][:-1, None] + torch.arange(m, device="cuda")).clamp_max(s["n"] - 1)
    q = s["q"].float()[row].reshape(c["seqs"], m, kvh, group, hd).transpose(1, 2).reshape(c["seqs"], kvh, m * group, hd)
    score = torch.matmul(q * s["scale"], k.transpose(-1, -2)).reshape(c["seqs"], kvh, m, group, s["max_kv"])
    pos = (s["kv_len"] - (s["row_start"][1:] - s["row_start"][:-1]))[:, None] + torch.arange(m, device="cuda")
    back = pos[:, :, None] - at
    seen = back >= 0
    if c["window"]:
        seen &= (back < c["window"]) | (at < c["sinks"])
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(c["seqs"], kvh, m * group, s["max_kv"]), v).reshape(c["seqs"], kvh, m, group, hd)
    out = (out / total).transpose(1, 2)
    return out.reshape(c["seqs"], m, c["heads"], hd)[s["row_seq"], s["row_at"]].to(s["out"].dtype)


def _pages_of(length, page):
    return torch.div(length + (page - 1), page, rounding_mode="floor")


def _plain_tables(s):
    page, before, rows = s["case"]["page"], s["kv_len"], s["new_rows"]
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    row_start = torch.cat((zero, rows.cumsum(0)))
    after = before + rows
    have, need = _pages_of(before, page), _pages_of(after, page)
    taken = torch.cat((zero, (need - have).cumsum(0)))  # pages taken in front of each sequence
    col = torch.arange(s["table"].shape[1], device="cuda")
    fresh = (col >= have[:, None]) & (col < need[:, None])
    nth = taken[:-1, None] + col - have[:, None]  # of the pages taken: from the end of the free list
    picked = s["free"][(s["free_count"] - 1 - nth).clamp(0, s["free"].shape[0] - 1)]
    table = torch.where(fresh, picked, s["table"])
    r = torch.arange(s["n"], device="cuda")
    b = (torch.searchsorted(row_start, r, right=True) - 1).clamp_max(rows.shape[0] - 1)
    there = r < row_start[-1]
    pos = torch.where(there, before[b] + r - row_start[b], -1)
    at = table[b, torch.div(pos, page, rounding_mode="floor").clamp_min(0)].long()
    slots = torch.where(there, at * page + pos % page, -1)
    # and back to the lengths to keep: the last page taken is the first to return
    count = s["free_count"] - taken[-1]
    back = (col >= _pages_of(s["keep"], page)[:, None]) & (col < need[:, None]) & (table >= 0)
    order = back.flatten().cumsum(0).reshape(back.shape)  # 1 for the first
    total = order[-1, -1]
    to = torch.where(back, count + total - order, s["free"].shape[0])
    free = torch.cat((s["free"], zero.to(torch.int32))).scatter(0, to.flatten(), table.flatten())[:-1]
    return {"row_start": row_start.to(torch.int32), "slots": slots, "positions": pos.to(torch.int32), "kv_len": torch.minimum(after, s["keep"]).to(torch.int32),
            "table": torch.where(back, -1, table), "free": free, "free_count": (count + total).to(torch.int32)}


def _plain_norm(s):
    x = s["block"].float()
    if s["post"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["post"]
    if s["gate"] is not None:
        x = x * s["gate"].float()
    r = s["residual"].float() + s["case"]["scale"] * x
    out = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * s["pre"]
    return {"residual": r.to(s["residual_out"].dtype), "out": out.to(s["out"].dtype)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "tables": _exact_tables, "norm": _exact_norm}[case["kind"]](case, s)


def _exact_norm(case, s):
    y, r = s["block"].double(), s["residual"].double()
    if case["post"]:
        y = y / torch.sqrt((y * y).sum(1, keepdim=True) / case["dim"] + EPS) * s["post"].double()
    r = r + case["scale"] * (y if case["gate"] == "none" else y * s["gate"].double())
    h = r / torch.sqrt((r * r).sum(1, keepdim=True) / case["dim"] + EPS)
    return {"residual": r, "out": h * s["pre"].double()}


def _exact_tables(case, s):
    """A list of free pages that pages are popped from, request by request, and put back on in the opposite order."""
    page = case["page"]
    table, kv, new, free = s["table"].tolist(), s["kv_len"].tolist(), s["new_rows"].tolist(), s["free"].tolist()
    count = int(s["free_count"])
    starts, slots, positions, popped = [0], [], [], []
    for b in range(len(kv)):
        for j in range(kv[b], kv[b] + new[b]):
            if j % page == 0:
                count -= 1
                table[b][j // page] = free[count]
                popped.append((b, j // page))
            slots.append(table[b][j // page] * page + j % page)
            positions.append(j)
        starts.append(len(slots))
    pad = [-1] * (s["n"] - len(slots))
    for b, i in reversed(popped):
        free[count], table[b][i] = table[b][i], -1
        count += 1
    return {"row_start": _ints(starts), "slots": _ints(slots + pad, torch.int64), "positions": _ints(positions + pad), "kv_len": _ints(kv), "table": _ints(table), "free": _ints(free),
            "free_count": _ints([count])}


def _cached(case, s, name, b, j):
    """Cached positions j of sequence b, in 64 bits: [position][kv head][hd]."""
    pg, off = s["table"][b].long()[torch.div(j, case["page"], rounding_mode="floor")], torch.remainder(j, case["page"])
    x = s[name][pg, off] if case["layout"] == "NHD" else s[name][pg, :, off]
    u = torch.empty((*x.shape[:-1], case["hd"]), dtype=torch.float64, device="cuda")
    u[..., 0::2], u[..., 1::2] = torch.remainder(x, 16).double(), torch.div(x, 16, rounding_mode="floor").double()
    pair = s[name + "_scale"][pg, :, off].double()
    return u * pair[:, :, :1] + pair[:, :, 1:]


def _exact_append(case, s):
    def turn(x, held):  # held: as a quantiser sees it, products and sum rounded to 32 bits one by one (a step's middle may lie between)
        half = x.shape[-1] // 2
        a, b, c, d = x[..., :half].double(), x[..., half:].double(), s["cos"][s["row_pos"]].double()[:, None], s["sin"][s["row_pos"]].double()[:, None]
        r = (lambda y: y.float().double()) if held else (lambda y: y)
        return torch.cat((r(r(a * c) - r(b * d)), r(r(a * d) + r(b * c))), -1)

    def bf16(x, up):  # the nearest bf16 number on one side
        near = x.to(torch.bfloat16).double()
        part, power = torch.frexp(near)  # near = part * 2^power, 0.5 <= |part| < 1
        unit = torch.exp2((power.clamp_min(-125) - 8).double())
        unit = torch.where((part.abs() == 0.5) & ((near > 0) != up), unit / 2, unit)
        return torch.where(near < x, near + unit, near) if up else torch.where(near > x, near - unit, near)

    k, v, q = s["new_k"].double(), s["new_v"].double(), None
    if case["rope"]:
        k, q = turn(s["new_k"], True), turn(s["q"], False)
    out = {"q": q}
    for name, x in (("k", k), ("v", v)):
        zero = bf16(x.min(-1, keepdim=True).values, False)
        step = bf16((x.max(-1, keepdim=True).values - zero) / 15, True)
        out[name] = zero + step * torch.round((x - zero).float().double() * (1 / step).float().double())  # (both as 32 bits hold them)
    return out


def _exact_attend(case, s):
    rows, kv = _lengths(case)
    starts = s["row_start"].tolist()
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros((s["n"], case["heads"], case["hd"]), dtype=torch.float64, device="cuda")
    for b in range(len(kv)):
        j = torch.arange(kv[b], device="cuda")
        k, v = _cached(case, s, "k", b, j), _cached(case, s, "v", b, j)
        for i0 in range(0, rows[b], 512):
            i1 = min(rows[b], i0 + 512)
            hi = kv[b] - rows[b] + i1
            p = torch.arange(hi - (i1 - i0), hi, device="cuda")[:, None]
            at = torch.arange(hi, device="cuda")[None]
            keep = at <= p
            if case["window"]:
                keep = keep & ((at > p - case["window"]) | (at < case["sinks"]))
            for h in range(case["kv_heads"]):
                qs = s["q"][starts[b] + i0:starts[b] + i1, h * group:(h + 1) * group].double()
                w = torch.einsum("igd,jd->gij", qs, k[:hi, h]) * s["scale"]
                w = torch.softmax(w.masked_fill(~keep, -math.inf), -1)
                out[starts[b] + i0:starts[b] + i1, h * group:(h + 1) * group] = torch.einsum("gij,jd->igd", w, v[:hi, h])
    return out

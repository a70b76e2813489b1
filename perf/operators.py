"""The paged KV cache and its attention, as cases that can be timed and compared: plain forms beside the library's calls.

A case is one of

* ``append``  new tokens' K and V written into their pages (and, with ``rope``, rotated on the way, the queries too); a cache in
              8 bits is read back in the same pass, as rows of 16 bits;
* ``read``    cached rows of every sequence gathered from their pages into contiguous rows;
* ``attend``  attention of the new tokens of every sequence (one, a few, a chunk, a whole prompt) over the cache.

A batch has ``seqs`` sequences.  ``chunks`` of them bring about ``new`` tokens each, the others one token; their cached lengths lie
between ``kv_min`` and ``kv_max`` (new tokens included) and are the same for every seed, so that the work of a case is known.
Pages are handed out in random order, as after some hours of serving.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
ROPE_LEN = 16384


def _case(kind, name=None, **kw):
    c = dict(kind=kind, seqs=1, chunks=0, new=1, kv_min=1, kv_max=1, heads=32, kv_heads=32, hd=128, page=16, io="bf16", cache="bf16",
             window=0, sinks=0, rope=False, layout="NHD")
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # A decode step of a small batch on the 7B shape: what the projections give (f32) is rotated and written; latency counts.
        _case("append", "append-step-7b-f16", seqs=16, kv_min=40, kv_max=2000, io="f32", cache="f16", rope=True),
        # A decode step of a large batch on the 70B shape with a cache in 8 bits, read back as a program does that checks or moves it.
        _case("append", "append-step-70b-i8", seqs=64, kv_min=1, kv_max=4000, heads=64, kv_heads=8, cache="i8"),
        # The chunks of several long prompts at once.
        _case("append", "append-chunks-13b-i8", seqs=6, chunks=6, new=1500, kv_min=1500, kv_max=6000, heads=40, kv_heads=40, page=32, cache="i8"),
        # One short sequence copied out (to another cache, or to the host).
        _case("read", "read-one-7b-f16", kv_min=333, kv_max=333, cache="f16", io="f16"),
        # A batch's whole caches copied out, ragged, 8 bits to 16.
        _case("read", "read-batch-70b-i8", seqs=48, kv_min=100, kv_max=8000, heads=64, kv_heads=8, cache="i8", page=64, layout="HND"),
        # One user, one token: the smallest call of serving.
        _case("attend", "attend-one-7b-f16", kv_min=517, kv_max=517, cache="f16", io="f16"),
        # A full serving batch, very ragged, grouped query heads, cache in 8 bits.
        _case("attend", "attend-step-70b-i8", seqs=64, kv_min=1, kv_max=8192, heads=64, kv_heads=8, cache="i8"),
        # Long streams with a bounded window and a few sinks.
        _case("attend", "attend-stream-13b-window", seqs=8, kv_min=20000, kv_max=60000, heads=40, kv_heads=40, page=32, window=4096, sinks=4),
        # Drafted tokens verified: five rows a sequence.
        _case("attend", "attend-verify-70b-bf16", seqs=12, chunks=12, new=5, kv_min=300, kv_max=3000, heads=64, kv_heads=8, page=16),
        # Serving with chunked prompts: two chunks among single tokens.
        _case("attend", "attend-mixed-13b-bf16", seqs=26, chunks=2, new=389, kv_min=30, kv_max=2500, heads=40, kv_heads=40),
        # The last chunk of a long document over a cache in 8 bits.
        _case("attend", "attend-chunk-70b-i8", chunks=1, new=512, kv_min=15000, kv_max=15000, heads=64, kv_heads=8, cache="i8", page=64),
        # A whole long prompt.
        _case("attend", "attend-prompt-7b-8191", chunks=1, new=8191, kv_min=8191, kv_max=8191, page=64, layout="HND"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    most = _cost(listed()[-1])
    while True:
        kv_heads, group = rng.choice([(32, 1), (40, 1), (8, 8), (8, 4), (4, 2), (2, 8), (1, 16), (4, 3), (16, 1)])
        kind = rng.choice(["append", "read", "attend", "attend", "attend", "attend"])
        cache = rng.choice(["f16", "bf16", "i8", "i8"])
        io = "bf16" if cache == "i8" else cache
        c = _case(kind, heads=kv_heads * group, kv_heads=kv_heads, hd=rng.choice([128, 128, 128, 64]), page=rng.choice([16, 32, 64, 128]),
                  io=io, cache=cache, layout=rng.choice(["NHD", "HND"]))
        c["seqs"] = _log(rng, 1, 128)
        c["kv_max"] = _log(rng, 2, 65536 if c["seqs"] < 8 else 8192)
        c["kv_min"] = rng.randint(1, c["kv_max"])
        if kind != "read" and rng.random() < 0.6:
            c["chunks"] = rng.randint(1, max(1, min(c["seqs"], 8)))
            c["new"] = _log(rng, 2, 8191)
            c["kv_max"] = max(c["kv_max"], c["new"] + 1)
        if kind == "append":
            c["rope"] = rng.random() < 0.5 and c["kv_max"] <= ROPE_LEN
            if c["rope"] and cache != "i8":
                c["io"] = rng.choice(["f32", io])
        if kind == "attend" and rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 16, 8192), rng.choice([0, 1, 4, 17, 64])
        if _cost(c) <= most and _plain_bytes(c) <= 30e9:
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
    kv = [max(a, b) for a, b in zip(kv, rows)]
    return (kv, kv) if case["kind"] == "read" else (rows, kv)


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
    caches = 2 * case["seqs"] * max(kv) * case["kv_heads"] * case["hd"] * 4
    return caches + (12 * case["seqs"] * max(rows) * case["heads"] * max(kv) if case["kind"] == "attend" else 0)


def _cost(case):
    """About what the plain form takes, in bytes moved."""
    w = work(case)
    return 4 * _plain_bytes(case) + w["bytes"] + (4 * case["hd"] * case["seqs"] * max(_lengths(case)[0]) * case["heads"] * max(_lengths(case)[1]) / 10 if case["kind"] == "attend" else 0)


def work(case):
    rows, kv = _lengths(case)
    row = case["kv_heads"] * case["hd"]
    held = 2 * (row * SIZE[case["cache"]] + (4 * case["kv_heads"] if case["cache"] == "i8" else 0))  # K and V of a cached token
    q_row = case["heads"] * case["hd"]
    if case["kind"] == "attend":
        pairs, keys = _pairs(case)
        return {"bytes": keys * held + 2 * sum(rows) * q_row * SIZE[case["io"]], "flops": 4.0 * case["hd"] * case["heads"] * pairs}
    n = sum(rows)
    if case["kind"] == "read":
        return {"bytes": n * (held + 2 * row * SIZE[case["io"]]), "flops": 0}
    back = 2 * n * row * 2 + n * held if case["cache"] == "i8" else 0
    queries = n * q_row * (SIZE[case["io"]] + 2) if case["rope"] else 0
    return {"bytes": n * (held + 2 * row * SIZE[case["io"]]) + queries + back, "flops": 0}


def _floats(gen, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(generator=gen) if dtype.is_floating_point else out.random_(-127, 128, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, kv = _lengths(case)
    n, page, kvh, hd = sum(rows), case["page"], case["kv_heads"], case["hd"]
    width = -(-max(kv) // page) + 1
    used = [-(-x // page) for x in kv]
    n_pages = sum(used) + 8
    order = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)[: sum(used)]
    seq = torch.repeat_interleave(torch.arange(len(used)), torch.tensor(used))
    first = torch.tensor([0] + used).cumsum(0)
    col = torch.arange(sum(used)) - first[seq]
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    table[seq.cuda(), col.cuda()] = order
    row_start = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    row_seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    s = {
        "case": case, "table": table, "row_start": row_start.cuda(), "kv_len": torch.tensor(kv, dtype=torch.int32).cuda(),
        "n": n, "max_rows": max(rows), "max_kv": max(kv), "scale": 1.0 / math.sqrt(hd),
        # where each row is: its sequence, its place in it and its position
        "row_seq": row_seq.cuda(), "row_at": (torch.arange(n) - row_start[row_seq]).cuda(),
        "row_pos": (torch.arange(n) - row_start[row_seq] + torch.tensor(kv)[row_seq] - torch.tensor(rows)[row_seq]).cuda(),
    }
    ctype, io = TYPES[case["cache"]], TYPES[case["io"]]
    shape = (n_pages, page, kvh, hd) if case["layout"] == "NHD" else (n_pages, kvh, page, hd)
    for x in "kv":
        s[x] = _floats(gen, shape, ctype)
        s[x + "_scale"] = torch.empty((n_pages, kvh, page), device="cuda").uniform_(0.01, 0.04, generator=gen) if ctype == torch.int8 else None
    rounded = TYPES["bf16"] if case["cache"] == "i8" else ctype  # the 16-bit type beside the cache
    if case["kind"] == "append":
        # channels differ in size, as keys' do
        channel = torch.empty((kvh, hd), device="cuda").normal_(generator=gen).mul_(0.7).exp_()
        s["new_k"] = (_floats(gen, (n, kvh, hd), torch.float32) * channel).to(io)
        s["new_v"] = _floats(gen, (n, kvh, hd), io)
        if case["rope"]:
            s["q"], s["q_out"] = _floats(gen, (n, case["heads"], hd), io), torch.empty((n, case["heads"], hd), dtype=rounded, device="cuda")
            angle = torch.arange(ROPE_LEN).double()[:, None] * 10000.0 ** (-torch.arange(hd // 2).double() / (hd // 2))
            s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
        s["k_back"], s["v_back"] = (torch.empty((n, kvh, hd), dtype=rounded, device="cuda") if case["cache"] == "i8" else None for _ in "kv")
    elif case["kind"] == "read":
        s["k_back"], s["v_back"] = (torch.empty((n, kvh, hd), dtype=io, device="cuda") for _ in "kv")
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
        return {"append": _own_append, "read": _own_read, "attend": _own_attend}[kind](s)
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[kind](s)


# ---- the library's calls -------------------------------------------------------------------------------------------------

def _own_append(s):
    rope = (s["cos"], s["sin"]) if s["case"]["rope"] else None
    s["pages"].append(s["batch"], s["new_k"], s["new_v"], rope=rope, q=s.get("q"), q_out=s.get("q_out"))
    if s["k_back"] is not None:
        s["pages"].read(s["batch"], s["k_back"], s["v_back"])
        return {"k": s["k_back"], "v": s["v_back"], "q": s.get("q_out")}
    return {"k": s["k"], "v": s["v"], "q": s.get("q_out")}


def _own_read(s):
    s["pages"].read(s["batch"], s["k_back"], s["v_back"])
    return {"k": s["k_back"], "v": s["v_back"]}


def _own_attend(s):
    c = s["case"]
    s["pages"].attend(s["batch"], s["q"], s["out"], scale=s["scale"], window=c["window"], sinks=c["sinks"], workspace=s["workspace"])
    return s["out"]


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
    if s["k_back"] is None:
        _pool(s, "k")[page, at], _pool(s, "v")[page, at] = k.to(s["k"].dtype), v.to(s["v"].dtype)
        return {"k": s["k"], "v": s["v"], "q": q}
    _quantise(s, "k", k, page, at)
    _quantise(s, "v", v, page, at)
    return {**_plain_read(s), "q": q}


def _quantise(s, name, x, page, at):
    most = x.abs().amax(-1, keepdim=True)
    _pool(s, name)[page, at] = torch.round(x * (127.0 / most)).to(torch.int8)
    s[name + "_scale"].transpose(1, 2)[page, at] = (most / 127.0)[..., 0]


def _plain_read(s):
    page, at = _slots(s)
    return {x: _values(s, x, page, at).to(s["k_back"].dtype) for x in "kv"}


def _values(s, name, page, at):
    x = _pool(s, name)[page, at].float()
    return x if s[name + "_scale"] is None else x * s[name + "_scale"].transpose(1, 2)[page, at][..., None]


def _plain_attend(s):
    c = s["case"]
    kvh, hd, page, group = c["kv_heads"], c["hd"], c["page"], c["heads"] // c["kv_heads"]
    # every sequence's keys and values, padded to the longest: [sequence][kv head][position][hd]
    at = torch.arange(s["max_kv"], device="cuda")
    pages = s["table"][:, at // page].long().clamp_min(0)
    k, v = (_values(s, x, pages, at % page).transpose(1, 2) for x in "kv")
    there = (at < s["kv_len"][:, None])[:, None, :, None]
    v = torch.where(there, v, torch.zeros((), device="cuda"))
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
    most = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(most == -math.inf, torch.zeros((), device="cuda"), most)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(c["seqs"], kvh, m * group, s["max_kv"]), v).reshape(c["seqs"], kvh, m, group, hd)
    out = torch.where(total > 0, out / total, torch.zeros((), device="cuda")).transpose(1, 2)
    return out.reshape(c["seqs"], m, c["heads"], hd)[s["row_seq"], s["row_at"]].to(s["out"].dtype)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    rows, kv = _lengths(case)
    page = case["page"]
    starts = s["row_start"].tolist()

    def cached(name, b, lo, hi):
        """Cached positions lo .. hi - 1 of sequence b, in 64 bits: [position][kv head][hd]."""
        j = torch.arange(lo, hi, device="cuda")
        pg, off = s["table"][b].long()[torch.div(j, page, rounding_mode="floor")], torch.remainder(j, page)
        x = s[name][pg, off] if case["layout"] == "NHD" else s[name][pg, :, off]
        x = x.double()
        return x * s[name + "_scale"][pg, :, off].double()[:, :, None] if s[name + "_scale"] is not None else x

    if case["kind"] == "read":
        return {x: torch.cat([cached(x, b, 0, kv[b]) for b in range(len(kv))]) for x in "kv"}

    def turn(x, pos):
        half = x.shape[-1] // 2
        z = torch.complex(x[..., :half].double(), x[..., half:].double())
        z = z * torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        return torch.cat((z.real, z.imag), -1)

    if case["kind"] == "append":
        k, v, q = s["new_k"].double(), s["new_v"].double(), None
        if case["rope"]:
            k, q = turn(s["new_k"], s["row_pos"]), turn(s["q"], s["row_pos"])
        if case["cache"] == "i8":
            step = {x: y.abs().max(-1, keepdim=True).values / 127 for x, y in (("k", k), ("v", v))}
            return {"k": torch.round(k / step["k"]) * step["k"], "v": torch.round(v / step["v"]) * step["v"], "q": q}
        pools = {}
        for name, x in (("k", k), ("v", v)):
            pool = s[name].double()
            for b in range(len(kv)):
                j = torch.arange(kv[b] - rows[b], kv[b], device="cuda")
                pg, off = s["table"][b].long()[torch.div(j, page, rounding_mode="floor")], torch.remainder(j, page)
                if case["layout"] == "NHD":
                    pool[pg, off] = x[starts[b]:starts[b + 1]]
                else:
                    pool[pg, :, off] = x[starts[b]:starts[b + 1]]
            pools[name] = pool
        return {**pools, "q": q}

    group = case["heads"] // case["kv_heads"]
    out = torch.zeros((s["n"], case["heads"], case["hd"]), dtype=torch.float64, device="cuda")
    for b in range(len(kv)):
        k, v = cached("k", b, 0, kv[b]), cached("v", b, 0, kv[b])
        for i0 in range(0, rows[b], 512):
            i1 = min(rows[b], i0 + 512)
            p0 = kv[b] - rows[b] + i0
            hi = kv[b] - rows[b] + i1
            p = torch.arange(p0, hi, device="cuda")[:, None]
            j = torch.arange(hi, device="cuda")[None]
            keep = j <= p
            if case["window"]:
                keep = keep & ((j > p - case["window"]) | (j < case["sinks"]))
            for h in range(case["kv_heads"]):
                qs = s["q"][starts[b] + i0:starts[b] + i1, h * group:(h + 1) * group].double()
                w = torch.einsum("igd,jd->gij", qs, k[:hi, h]) * s["scale"]
                w = torch.softmax(w.masked_fill(~keep, -math.inf), -1)
                out[starts[b] + i0:starts[b] + i1, h * group:(h + 1) * group] = torch.einsum("gij,jd->igd", w, v[:hi, h])
    return out

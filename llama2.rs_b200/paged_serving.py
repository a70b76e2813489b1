"""Several sequences through one attention layer with a paged cache: quantised projections, RoPE, 4-bit, int8 or f16 pages, chunked prompts among single tokens.

    python llama2.rs_b200/paged_serving.py                                   # 7B heads, int8 pages, 16 sequences
    python llama2.rs_b200/paged_serving.py --heads 64 --kv-heads 8 --cache f16 --window 1024 --sinks 4
    python llama2.rs_b200/paged_serving.py --cache u4 --tables device        # pages handed out on the GPU

A step takes up to --budget rows: one of every sequence that is past its prompt, the rest of the room for prompts, in order.  Pages are handed out as
sequences grow and given back when these end and, with a window, when no row can see them any more: by lists of this program, whose tables are copied to the GPU in
every step, or (--tables device) by l2_kv_plan and l2_kv_release, with tables that never leave it.  There is no model behind the layer: a prompt is random rows, and the
next row of a sequence is the layer's own (normalised) output for the row before.  Weights are random in the checkpoint's layout; RoPE is that of the
package's models (--rotation pairs: of plain pairs, for weights that want it).
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


class PagedLayer:
    """wq / wk / wv -> RoPE, append -> attend -> wo on device tensors; the cache's pages and who has them.  rotation: "pairs", or "model" as the package's
    models do it, for their weights."""

    def __init__(self, dim, heads, kv_heads, *, cache="i8", n_pages=512, page_size=32, positions=4096, window=0, sinks=0, group_size=64, seed=0, weights=None, rotation="pairs"):
        import torch
        import llama2_rs as l2
        from qlinear_bench import random_qlinear
        self.l2, self.torch = l2, torch
        self.dim, self.heads, self.kv_heads, self.hd = dim, heads, kv_heads, 128
        self.window, self.sinks, self.page_size = window, sinks, page_size
        rng = np.random.default_rng(seed)
        shapes = {"q": (dim, heads * 128), "k": (dim, kv_heads * 128), "v": (dim, kv_heads * 128), "o": (heads * 128, dim)}
        self.weights = weights or {n: random_qlinear(rng, i, o, group_size) for n, (i, o) in shapes.items()}
        self.linear = {n: l2.QLinear(*w, group_size) for n, w in self.weights.items()}
        kind = {"u4": torch.uint8, "i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}[cache]
        k, v = (torch.zeros((n_pages, page_size, kv_heads, 64 if cache == "u4" else 128), dtype=kind, device="cuda") for _ in "kv")
        scales = []
        if cache == "i8":
            scales = [torch.zeros((n_pages, kv_heads, page_size), device="cuda") for _ in "kv"]
        if cache == "u4":
            scales = [torch.zeros((n_pages, kv_heads, page_size, 2), dtype=torch.bfloat16, device="cuda") for _ in "kv"]
        self.pages = l2.KvPages(k, v, *scales)
        self.q_type = torch.float16 if cache == "f16" else torch.bfloat16
        self.rope, self.rotation = l2.KvRope(positions), rotation
        self.free = list(range(n_pages))[::-1]
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def _project(self, name, x):
        out = self.torch.empty((x.shape[0], self.linear[name].out_features), device="cuda")
        self.linear[name].matvec_dev(x.data_ptr(), out.data_ptr(), x.shape[0], self.torch.cuda.current_stream().cuda_stream)
        return out

    def pages_for(self, sequence, rows):
        """Pages that a sequence needs besides its own for so many more rows."""
        return max(0, -(-(sequence["length"] + rows) // self.page_size) - len(sequence["table"]))

    def release(self, sequence):
        """Gives back the pages of a sequence that has ended.  (Work enqueued before is in front of what their next owner enqueues.)"""
        self.free += [page for page in sequence["table"] if page >= 0]
        sequence["table"], sequence["length"] = [], 0

    def step(self, x, sequences, rows):
        """x [rows in all, dim] f32, rows[i] new rows of sequences[i] (dicts with `length` and `table`): the layer's output, f32."""
        torch, n = self.torch, x.shape[0]
        new = [self.pages_for(s, r) for s, r in zip(sequences, rows)]
        if sum(new) > len(self.free):
            raise RuntimeError("%d pages needed, %d left" % (sum(new), len(self.free)))
        for s, r, pages in zip(sequences, rows, new):
            s["length"] += r
            s["table"] += [self.free.pop() for _ in range(pages)]
        width = max(len(s["table"]) for s in sequences)
        table = torch.tensor([s["table"] + [-1] * (width - len(s["table"])) for s in sequences], dtype=torch.int32).cuda()
        kv_len = torch.tensor([s["length"] for s in sequences], dtype=torch.int32).cuda()
        start = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32).cuda()
        batch = self.l2.KvBatch(table, kv_len, start, n, max(rows), status=self.status)
        out = self._attention(batch, x, torch.empty)
        if self.window:  # pages that no later row sees
            for s in sequences:
                for i in range(-(-self.sinks // self.page_size), max(0, s["length"] - self.window + 1) // self.page_size):
                    if s["table"][i] >= 0:
                        self.free.append(s["table"][i])
                        s["table"][i] = -1
        return self._project("o", out)

    def _attention(self, batch, x, room):
        """room: torch.empty where every row is a sequence's, else torch.zeros."""
        n = x.shape[0]
        q, k, v = (self._project(name, x) for name in "qkv")
        q16 = room((n, self.heads, 128), dtype=self.q_type, device="cuda")
        self.pages.append(batch, k.view(n, -1, 128), v.view(n, -1, 128), rope=self.rope, rotation=self.rotation, q=q.view(n, -1, 128), q_out=q16)
        out = self.pages.attend(batch, q16, room((n, self.heads, 128), device="cuda"), window=self.window, sinks=self.sinks)
        return out.view(n, -1)

    def normed(self, y):
        """The rows' next inputs."""
        return self.l2.block_norm(y, None, self.torch.empty_like(y))[1]


class PlannedLayer(PagedLayer):
    """The same with the tables, the lengths and the free pages of up to `n_seqs` sequences on the device: the host says how many rows each brings, and which have ended."""

    def __init__(self, *args, n_seqs, budget, positions=4096, n_pages=512, page_size=32, **kw):
        super().__init__(*args, positions=positions, n_pages=n_pages, page_size=page_size, **kw)
        torch = self.torch
        ints = lambda *shape, fill=0: torch.full(shape, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.lengths, self.row_start = ints(n_seqs, -(-positions // page_size), fill=-1), ints(n_seqs), ints(n_seqs + 1)
        self.free_pages, self.free_count = torch.arange(n_pages, dtype=torch.int32, device="cuda"), ints(1, fill=n_pages)
        self.tables = self.l2.KvTables(self.table, self.lengths, self.free_pages, self.free_count, page_size, status=self.status)
        self.n_seqs, self.budget = n_seqs, budget

    def step_planned(self, x, rows):
        """x [rows in all, dim] f32, rows[b] of them of sequence b, one after the other: the layer's output, f32."""
        n, torch = x.shape[0], self.torch
        if n > self.budget:
            raise ValueError("%d rows, of %d" % (n, self.budget))
        self.tables.plan(torch.tensor(rows, dtype=torch.int32).cuda(), self.row_start, n, max(rows))
        out = self._attention(self.l2.KvBatch(self.table, self.lengths, self.row_start, n, max(rows), status=self.status), x, torch.zeros)  # (a step without room leaves all rows out)
        if self.window:
            self.tables.release(window=self.window, sinks=self.sinks)
        return self._project("o", out)

    def end(self, sequences):
        """Gives back the pages of sequences (indices) that have ended."""
        keep = [1 << 30] * self.n_seqs
        for b in sequences:
            keep[b] = 0
        self.tables.release(self.torch.tensor(keep, dtype=self.torch.int32).cuda())


def serve_planned(layer, prompts, tokens, budget):
    """As serve, by a PlannedLayer.  The status word is looked at where sequences end, before their outputs count for anything: a RuntimeError says what it
    holds (pages that ran out, ..), and the pages of all sequences have gone back."""
    torch = layer.torch
    seqs = [{"todo": p, "out": [], "left": tokens} for p in prompts]
    steps = total = 0
    while any(len(s["todo"]) or s["left"] > 0 for s in seqs):
        room, rows, xs, ended = budget, [0] * layer.n_seqs, {}, []
        for b in sorted((b for b, s in enumerate(seqs) if len(s["todo"]) or s["left"] > 0), key=lambda b: len(seqs[b]["todo"]) > 1):  # single rows first
            s = seqs[b]
            r = rows[b] = min(room, len(s["todo"]) or 1)
            if r == 0:
                break
            if len(s["todo"]):
                xs[b] = s["todo"][:r]
            else:
                xs[b] = layer.normed(s["out"][-1][-1:])
                s["left"] -= 1
            s["todo"] = s["todo"][r:]
            room -= r
        y = layer.step_planned(torch.cat([xs[b] for b in sorted(xs)]), rows)
        for b, part in zip(sorted(xs), y.split([rows[b] for b in sorted(xs)])):
            seqs[b]["out"].append(part)
            if not len(seqs[b]["todo"]) and seqs[b]["left"] <= 0:
                ended.append(b)
        if ended:
            status = int(layer.status)
            layer.end(range(len(seqs)) if status else ended)
            if status:
                raise RuntimeError("a step went wrong: status %d" % status)
        steps, total = steps + 1, total + sum(rows)
    return [torch.cat(s["out"]) for s in seqs], steps, total


def serve(layer, prompts, tokens, budget):
    """Runs every prompt ([n, dim] rows) and then `tokens` rows of its own: (all outputs of each sequence, steps, rows)."""
    torch = layer.torch
    seqs = [{"length": 0, "table": [], "todo": p, "out": [], "left": tokens} for p in prompts]
    steps = total = 0
    while any(len(s["todo"]) or s["left"] > 0 for s in seqs):
        room, picked, rows, xs = budget, [], [], []
        for s in sorted((s for s in seqs if len(s["todo"]) or s["left"] > 0), key=lambda s: len(s["todo"]) > 1):  # single rows first
            r = min(room, len(s["todo"]) or 1)
            if r == 0:
                break
            x = s["todo"][:r] if len(s["todo"]) else None
            if x is None:  # past its prompt: the row before it, normalised, goes in again
                x = layer.normed(s["out"][-1][-1:])
                s["left"] -= 1
            s["todo"] = s["todo"][r:]
            picked.append(s), rows.append(r), xs.append(x)
            room -= r
        y = layer.step(torch.cat(xs), picked, rows)
        for s, part in zip(picked, y.split(rows)):
            s["out"].append(part)
            if not len(s["todo"]) and s["left"] <= 0:
                layer.release(s)
        steps, total = steps + 1, total + sum(rows)
    return [torch.cat(s["out"]) for s in seqs], steps, total


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=32)
    ap.add_argument("--cache", choices=["u4", "i8", "f16", "bf16"], default="i8")
    ap.add_argument("--tables", choices=["host", "device"], default="host", help="who hands out pages")
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--sequences", type=int, default=16)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--budget", type=int, default=512)
    ap.add_argument("--rotation", choices=["model", "pairs"], default="model", help="RoPE as the package's models do it, or of plain pairs")
    args = ap.parse_args()
    import torch
    if not torch.cuda.is_available():
        raise SystemExit("paged_serving needs a GPU: there is no CPU path")
    more = {"n_seqs": args.sequences, "budget": args.budget} if args.tables == "device" else {}
    layer = (PlannedLayer if more else PagedLayer)(args.heads * 128, args.heads, args.kv_heads, cache=args.cache, window=args.window, sinks=args.sinks, n_pages=2048, rotation=args.rotation, **more)
    run = serve_planned if more else serve
    rng = np.random.default_rng(1)
    prompts = [torch.randn(int(n), layer.dim, device="cuda") for n in rng.integers(5, 900, args.sequences)]
    run(layer, prompts, 2, args.budget)  # the layers' buffers, the kernels' first launches
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    outs, steps, rows = run(layer, prompts, args.tokens, args.budget)
    end.record()
    torch.cuda.synchronize()
    if int(layer.status):
        raise SystemExit("status %d" % int(layer.status))
    ms = begin.elapsed_time(end)
    print("%d sequences, %d rows in %d steps: %.1f ms, %.0f rows/s, largest output %.3g" % (len(outs), rows, steps, ms, rows / ms * 1e3, max(float(o.abs().max()) for o in outs)))


if __name__ == "__main__":
    main()

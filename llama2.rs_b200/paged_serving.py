"""Several sequences through one attention layer with a paged cache: quantised projections, RoPE, int8 or f16 pages, chunked prompts among single tokens.

    python llama2.rs_b200/paged_serving.py                                   # 7B heads, int8 pages, 16 sequences
    python llama2.rs_b200/paged_serving.py --heads 64 --kv-heads 8 --cache f16 --window 1024 --sinks 4

A step takes up to --budget rows: one of every sequence that is past its prompt, the rest of the room for prompts, in order.  Pages are handed out as
sequences grow and given back when these end and, with a window, when no row can see them any more.  There is no model behind the layer: a prompt is random rows, and the
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
        kind = {"i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}[cache]
        k, v = (torch.zeros((n_pages, page_size, kv_heads, 128), dtype=kind, device="cuda") for _ in "kv")
        scales = [torch.zeros((n_pages, kv_heads, page_size), device="cuda") for _ in "kv"] if cache == "i8" else []
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
        q, k, v = (self._project(name, x) for name in "qkv")
        q16 = torch.empty((n, self.heads, 128), dtype=self.q_type, device="cuda")
        self.pages.append(batch, k.view(n, -1, 128), v.view(n, -1, 128), rope=self.rope, rotation=self.rotation, q=q.view(n, -1, 128), q_out=q16)
        out = self.pages.attend(batch, q16, torch.empty((n, self.heads, 128), device="cuda"), window=self.window, sinks=self.sinks)
        if self.window:  # pages that no later row sees
            for s in sequences:
                for i in range(-(-self.sinks // self.page_size), max(0, s["length"] - self.window + 1) // self.page_size):
                    if s["table"][i] >= 0:
                        self.free.append(s["table"][i])
                        s["table"][i] = -1
        return self._project("o", out.view(n, -1))


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
                y = s["out"][-1][-1:]
                x = y / (y.square().mean() + 1e-5).sqrt()
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
    ap.add_argument("--cache", choices=["i8", "f16", "bf16"], default="i8")
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
    layer = PagedLayer(args.heads * 128, args.heads, args.kv_heads, cache=args.cache, window=args.window, sinks=args.sinks, n_pages=2048, rotation=args.rotation)
    rng = np.random.default_rng(1)
    prompts = [torch.randn(int(n), layer.dim, device="cuda") for n in rng.integers(5, 900, args.sequences)]
    serve(layer, prompts, 2, args.budget)  # the layers' buffers, the kernels' first launches
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    outs, steps, rows = serve(layer, prompts, args.tokens, args.budget)
    end.record()
    torch.cuda.synchronize()
    if int(layer.status):
        raise SystemExit("status %d" % int(layer.status))
    ms = begin.elapsed_time(end)
    print("%d sequences, %d rows in %d steps: %.1f ms, %.0f rows/s, largest output %.3g" % (len(outs), rows, steps, ms, rows / ms * 1e3, max(float(o.abs().max()) for o in outs)))


if __name__ == "__main__":
    main()

"""The paged cache and its attention in 64 bits, position by position, for the tests."""
import math

import torch

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a unit in the last place, relative
# what the smallest subnormal numbers of a type leave out
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}


class Case:
    """A pool of pages in random order, and a step: rows[b] new rows of sequence b, which holds kv[b] positions."""

    def __init__(self, rows, kv, *, kv_heads=2, group=1, hd=128, page=16, cache=torch.float16, layout="NHD", seed=0, spare_rows=0, fill=1.0, n_pages=None):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.kv, self.kv_heads, self.group, self.hd, self.page, self.layout = list(rows), list(kv), kv_heads, group, hd, page, layout
        self.heads = kv_heads * group
        used = [-(-x // page) for x in kv]
        self.n_pages = n_pages or sum(used) + 3
        width = max(used + [1]) + 1
        order = torch.randperm(self.n_pages, generator=g)
        self.table = torch.full((len(kv), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n].int()
            at += n
        self.row_start = torch.tensor([0] + self.rows).cumsum(0).int()
        self.n = int(self.row_start[-1]) + spare_rows
        shape = (self.n_pages, page, kv_heads, hd) if layout == "NHD" else (self.n_pages, kv_heads, page, hd)
        gd = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.scales = [None, None]
        if cache == torch.int8:
            self.k, self.v = (torch.randint(-127, 128, shape, generator=gd, dtype=torch.int8, device="cuda") for _ in "kv")
            self.scales = [torch.empty((self.n_pages, kv_heads, page), device="cuda").uniform_(0.005, 0.03, generator=gd) * fill for _ in "kv"]
        else:
            self.k, self.v = (torch.randn(shape, generator=gd, device="cuda").mul_(fill).to(cache) for _ in "kv")
        self.device_arrays()

    def device_arrays(self):
        self.d_table, self.d_kv, self.d_start = self.table.cuda(), torch.tensor(self.kv, dtype=torch.int32).cuda(), self.row_start.cuda()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def handles(self, l2, **kw):
        pages = l2.KvPages(self.k, self.v, *self.scales, layout=self.layout)
        return pages, l2.KvBatch(self.d_table, self.d_kv, self.d_start, self.n, kw.get("max_rows", max(self.rows + [0])), status=self.status)

    def slot(self, b, j):
        return int(self.table[b, j // self.page]), j % self.page

    def at(self, t, page, off):
        """[kv_heads, hd] (or [kv_heads]) of a pool tensor (or scales, always [page, head, position])."""
        if t.dim() == 3:
            return t[page, :, off]
        return t[page, off] if self.layout == "NHD" else t[page, :, off]

    def cached(self, which, b):
        """Positions 0 .. kv[b] - 1 in 64 bits, [position, kv_heads, hd]."""
        j = torch.arange(self.kv[b])
        pages, offs = self.table[b].long()[j // self.page].cuda(), (j % self.page).cuda()
        x = self.at((self.k, self.v)[which], pages, offs).double()
        s = self.scales[which]
        return x if s is None else x * s[pages, :, offs].double()[..., None]


def attend(case, q, scale, window=0, sinks=0, p_unit=None):
    """(result, bound) [rows, heads, hd] in 64 bits.  The bound is on what l2_kv_attend may differ by before its result is rounded to out's type:
    a probability is rounded once (p_unit); a score is a sum of hd exact products in f32 and a product, the largest score likewise, and their
    difference goes through an exponential (relative error 2^-17 allowed for) whose argument is rounded; sums over T positions are in f32."""
    u = 2.0**-24
    p_unit = UNIT[q.dtype] if p_unit is None else p_unit
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for b, (n, kv) in enumerate(zip(case.rows, case.kv)):
        k, v = case.cached(0, b), case.cached(1, b)
        for i in range(n):
            r, p = int(case.row_start[b]) + i, kv - n + i
            if p < 0:
                continue
            j = torch.arange(p + 1, device="cuda")
            if window:
                j = j[(p - j < window) | (j < sinks)]
            for h in range(case.kv_heads):
                hs = slice(h * case.group, (h + 1) * case.group)
                kk, vv, qq = k[j, h], v[j, h], q[r, hs].double()
                s = qq @ kk.T * scale
                w = torch.softmax(s, -1)
                want[r, hs] = w @ vv
                size = (qq.abs() @ kk.abs().T * scale).amax(-1, keepdim=True)
                score = (case.hd + 4) * u * size
                rel = p_unit + 2 * score * math.log(2) * 1.5 + 4 * size * u + 2.0**-17 + (len(j) + 64) * u
                bound[r, hs] = rel * (w @ vv.abs())
    return want, bound


def check(got, want, bound, what=""):
    """got within bound of want, its own rounding on top; not finite where want is not."""
    t = got.dtype
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    room = bound + UNIT[t] * (want.abs() + bound) + TINY[t]
    bad = ~same & ~((got - want).abs() <= room)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its room at %s" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / room)[bad].nan_to_num(math.inf).max()), bad.nonzero()[0].tolist())

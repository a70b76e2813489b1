"""The paged cache in 4 bits in 64 bits, position by position, for the tests."""
import math

import numpy as np
import torch

from paged_reference import Case


class Case4(Case):
    """A pool of pages in 4 bits: k and v uint8 [.., hd / 2], scales [page, head, position, 2] bf16 (scale, zero)."""

    def __init__(self, rows, kv, *, low=0.01, high=0.3, **kw):
        super().__init__(rows, kv, cache=torch.int8, **kw)
        g = torch.Generator(device="cuda").manual_seed(kw.get("seed", 0) + 7)
        shape = (*self.k.shape[:-1], self.hd // 2)
        self.k, self.v = (torch.randint(0, 256, shape, generator=g, dtype=torch.uint8, device="cuda") for _ in "kv")
        self.scales = []
        for _ in "kv":
            pair = torch.empty((self.n_pages, self.kv_heads, self.page, 2), device="cuda").uniform_(0, 1, generator=g)
            pair[..., 0] = low + (high - low) * pair[..., 0]
            pair[..., 1] = -15 * pair[..., 1] * pair[..., 0]
            self.scales.append(pair.to(torch.bfloat16))

    def numbers(self, which, b):
        """(u, scale, zero) of positions 0 .. kv[b] - 1 in 64 bits: [position, kv_heads, hd] and [position, kv_heads, 1] twice."""
        j = torch.arange(self.kv[b])
        pages, offs = self.table[b].long()[j // self.page].cuda(), (j % self.page).cuda()
        x = self.at((self.k, self.v)[which], pages, offs)
        u = torch.stack((x & 15, x >> 4), -1).flatten(-2).double()
        pair = self.scales[which][pages, :, offs].double()
        return u, pair[..., :1], pair[..., 1:]

    def cached(self, which, b):
        u, scale, zero = self.numbers(which, b)
        return zero + scale * u


def attend4(case, q, scale, window=0, sinks=0, many=False, wide=None):
    """(result, bound) [rows, heads, hd] in 64 bits; the bound is on what l2_kv_attend may differ by before its result is rounded to out's type.

    Few rows: a score is a sum of hd exact products, a product with the position's scale, and the product of its zero and a sum of q: in f32, relative to the sum of
    their sizes; bf16 queries are resolved to 2^-39 of the row's largest.  A probability times a scale is rounded to f16, or to 2^-31 of the largest such product.
    Many rows: K, V and the probabilities are rounded to f16 (bf16 queries are resolved as above); to bf16, f16 queries too, if some row sees a pair that
    f16 does not hold: values beyond 65504, or steps below 2^-16.  A probability has f16's absolute step too, 2^-32 of the largest.
    The exponential: relative error 2^-17 allowed for; its argument is rounded; sums over T positions are in f32."""
    u1 = 2.0**-24
    wide = many and (not held(case, window, sinks) if wide is None else wide)
    unit = 2.0**-8 if wide else 2.0**-11
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for b, (n, kv) in enumerate(zip(case.rows, case.kv)):
        (ku, ks, kz), (vu, vs, vz) = case.numbers(0, b), case.numbers(1, b)
        for i in range(n):
            r, p = int(case.row_start[b]) + i, kv - n + i
            if p < 0:
                continue
            j = torch.arange(p + 1, device="cuda")
            if window:
                j = j[(p - j < window) | (j < sinks)]
            for h in range(case.kv_heads):
                hs = slice(h * case.group, (h + 1) * case.group)
                k, v, qq = (kz + ks * ku)[j, h], (vz + vs * vu)[j, h], q[r, hs].double()
                s = qq @ k.T * scale
                w = torch.softmax(s, -1)
                want[r, hs] = w @ v
                parts = (kz.abs() + ks.abs() * ku)[j, h]
                size = (qq.abs() @ parts.T * scale).amax(-1, keepdim=True)
                score = (case.hd + 8) * u1 * size
                if q.dtype == torch.bfloat16:
                    score = score + case.hd * 2.0**-39 * scale * (qq.abs().amax(-1, keepdim=True) * 15 * ks[j, h].abs().amax())
                p_unit = 2.0**-11
                if many:
                    rounded = unit * k.abs() + (0 if wide else 2.0**-25)
                    if wide and q.dtype == torch.float16:
                        rounded = rounded + 1.01 * unit * k.abs()
                    score = score + (qq.abs() @ rounded.T * scale).amax(-1, keepdim=True)
                    p_unit = 2 * unit + unit**2
                rel = p_unit + 2 * score * math.log(2) * 1.5 + 4 * size * u1 + 2.0**-17 + (len(j) + 64) * u1
                weight = w * vs[j, h].abs()[:, 0]
                bound[r, hs] = rel * (w @ (vz.abs() + vs.abs() * vu)[j, h]) + 15 * len(j) * 2.0**-31 * weight.amax(-1, keepdim=True)
                if many and not wide:
                    bound[r, hs] += 2.0**-25 + len(j) * 2.0**-32 * w.amax(-1, keepdim=True) * v.abs().amax()
    return want, bound


def held(case, window, sinks):
    """Whether f16 holds the values of every pair that some row sees."""
    for b, (n, kv) in enumerate(zip(case.rows, case.kv)):
        j, lo, hi = torch.arange(kv, device="cuda"), kv - n, kv - 1
        if n == 0 or hi < 0:
            continue
        seen = (j <= hi) & ((j > lo - window) | (j < sinks) if window else j >= 0)
        for which in (0, 1):
            _, s, z = (t[seen].abs() for t in case.numbers(which, b))
            ok = (z + 15 * s <= 65504) & ((s >= 2.0**-16) | ((s == 0) & ((z == 0) | (z >= 2.0**-14))))
            if not ok.all():
                return False
    return True


def quantise(x):
    """(u, scale, zero) of rows x [.., hd] (numpy f32), as the header defines them: integers and f32 numbers that bf16 holds."""
    x = np.asarray(x, np.float32)
    f32 = np.float32

    def floor16(v):  # the bf16 number at or below
        bits = np.asarray(v, f32).view(np.int32)
        down = (bits & ~0xffff).view(f32)  # towards zero
        return np.where(down > v, ((bits & ~0xffff) + 0x10000).view(f32), down).astype(f32)

    with np.errstate(all="ignore"):
        zero = floor16(x.min(-1, keepdims=True))
        span = (x.max(-1, keepdims=True) - zero).astype(f32)
        good = np.isfinite(x).all(-1, keepdims=True) & np.isfinite(span)
        exact = np.where(good, span, 1).astype(np.float64) / 15
        step = floor16(exact.astype(f32))
        for _ in range(3):  # the least with 15 scale >= span (from below: the division may have been rounded up)
            lower = (step.view(np.int32) - 0x10000).view(f32)
            step = np.where((lower.astype(np.float64) * 15 >= span) & (lower > 0), lower, step)
            step = np.where(step.astype(np.float64) * 15 < span, (step.view(np.int32) + 0x10000).view(f32), step)
        flat = span < f32(2.0**-100)
        inv = np.where(flat, f32(0), f32(1) / np.where(flat, f32(1), step)).astype(f32)
        u = np.rint((x - zero).astype(f32).astype(np.float64) * inv.astype(np.float64))
        nan = f32("nan")
        return np.where(good, u, 0), np.where(good, np.where(flat, f32(0), step), nan), np.where(good, zero, nan)

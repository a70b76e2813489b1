"""The paged KV cache in 4 bits (append, read back) and its attention against the same in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged4_reference import Case4, attend4, quantise  # noqa: E402
from paged_reference import check  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def run_attend(l2, c, io, *, scale=None, window=0, sinks=0, out_type=None, q=None, seed=5, max_rows=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if q is None:
        q = torch.randn((c.n, c.heads, c.hd), generator=g, device="cuda").to(io)
    out = torch.full((c.n, c.heads, c.hd), 7.0, dtype=out_type or io, device="cuda")
    pages, batch = c.handles(l2, **({"max_rows": max_rows} if max_rows else {}))
    pages.attend(batch, q, out, scale=scale, window=window, sinks=sinks)
    torch.cuda.synchronize()
    return q, out


def compare(l2, c, io, *, window=0, sinks=0, out_type=None, scale=None, what="", **kw):
    q, out = run_attend(l2, c, io, window=window, sinks=sinks, out_type=out_type, scale=scale, **kw)
    few = max(kw.get("max_rows") or 0, max(c.rows)) * c.group <= 16
    want, bound = attend4(c, q, scale or c.hd ** -0.5, window, sinks, many=not few)
    n = int(c.row_start[-1])
    check(out[:n], want[:n], bound[:n], what)
    assert (out[n:] == 7.0).all()  # rows of no sequence are left alone
    assert int(c.status) == 0


# ---- append and read -----------------------------------------------------------------------------------------------------

def stored(c, which, b, j):
    """(u [kv_heads, hd], scale, zero [kv_heads]) of a position, as numpy f32."""
    page, off = c.slot(b, j)
    x = c.at((c.k, c.v)[which], page, off).cpu().numpy()
    pair = c.scales[which][page, :, off].float().cpu().numpy()
    return np.stack((x & 15, x >> 4), -1).reshape(x.shape[0], -1), pair[:, 0], pair[:, 1]


def values(u, scale, zero, dtype):
    """zero + scale u, rounded to 32 bits and then to the type."""
    exact = zero.astype(np.float64)[..., None] + scale.astype(np.float64)[..., None] * u
    return torch.from_numpy(exact.astype(np.float32)).to(dtype)


@pytest.mark.parametrize("rope", [None, "pairs", "model"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("io", [F32, F16, BF16])
def test_append_and_read(l2, io, layout, hd, rope):
    for rows, kv in (([1, 1, 0, 1], [1, 33, 5, 64]), ([70, 1, 300, 5], [90, 7, 300, 3]), ([1], [1])):
        c = Case4(rows, kv, kv_heads=3, hd=hd, layout=layout, spare_rows=2)
        g = torch.Generator(device="cuda").manual_seed(3)
        k, v = (torch.randn((c.n, 3, hd), generator=g, device="cuda").to(io) for _ in "kv")
        q = torch.randn((c.n, 6, hd), generator=g, device="cuda").to(io)
        q_out = torch.full((c.n, 6, hd), 7.0, dtype=BF16, device="cuda")
        before = [t.clone() for t in (c.k, c.v, *c.scales)]
        angle = torch.rand((400, hd // 2), generator=g, device="cuda") * 6
        cos, sin = angle.cos(), angle.sin()
        pages, batch = c.handles(l2)
        pages.append(batch, k, v, rope=(cos, sin) if rope else None, rotation=rope, q=q, q_out=q_out)
        back = {t: [torch.full((c.n, 3, hd), 7.0, dtype=t, device="cuda") for _ in "kv"] for t in (F32, F16, BF16)}
        for t in back:
            pages.read(batch, *back[t])
        torch.cuda.synchronize()
        assert int(c.status) == 0
        hk, hv, hq = (t.float().cpu().numpy() for t in (k, v, q))
        co, si = cos.cpu().numpy(), sin.cpu().numpy()

        def turned(x, p):  # in 32 bits, rounded one by one
            if rope is None:
                return x
            a, b = x[..., :hd // 2], x[..., hd // 2:]
            first = a * co[p] - b * si[p]
            return np.concatenate((first, b * co[p] + (first if rope == "model" else a) * si[p]), -1).astype(np.float32)

        touched = torch.zeros((c.n_pages, c.page), dtype=torch.bool, device="cuda")
        for b in range(len(rows)):
            for i in range(rows[b]):
                r, p = int(c.row_start[b]) + i, kv[b] - rows[b] + i
                if p < 0:  # more rows than positions: nothing is written
                    assert all((back[t][w][r] == 7.0).all() for t in back for w in (0, 1)) and (q_out[r] == 7.0).all()
                    continue
                touched[c.slot(b, p)] = True
                assert torch.equal(q_out[r].cpu(), torch.from_numpy(turned(hq[r], p)).to(BF16))
                for w, x in ((0, turned(hk[r], p)), (1, hv[r])):
                    want, got = quantise(x), stored(c, w, b, p)
                    assert np.array_equal(got[1], want[1][:, 0]) and np.array_equal(got[2], want[2][:, 0]) and np.array_equal(got[0], want[0])
                    for t in back:
                        assert torch.equal(back[t][w][r].cpu(), values(*got, t))
                    assert (np.abs(values(*got, F32).numpy() - x) <= got[1][:, None] * 0.5001).all()
        assert all((back[t][w][int(c.row_start[-1]):] == 7.0).all() for t in back for w in (0, 1))
        for now, was, head in zip((c.k, c.v, *c.scales), before, (2, 2, 1, 1) if layout == "NHD" else (1, 1, 1, 1)):  # nothing else is written
            assert ((now == was).all(-1).all(head) | touched).all()


def test_rows_at_the_edges_of_what_numbers_hold(l2):
    """Equal elements, tiny and huge spans, elements next to the middle of a step, values that are not finite."""
    big = 3.0e38
    rows = [np.zeros(128), np.full(128, 5.3), np.full(128, -5.3), np.linspace(-1, 1, 128), np.linspace(100, 101, 128), np.linspace(0, 15, 128), np.arange(128) % 31 / 2.0,
            np.linspace(-2.0**-110, 2.0**-110, 128), np.linspace(0, 2.0**-99, 128), np.linspace(-1e30, 1e30, 128), np.linspace(0, big, 128), np.linspace(-big, big, 128),
            np.where(np.arange(128) == 3, np.nan, 1.0), np.where(np.arange(128) == 70, np.inf, 1.0), np.where(np.arange(128) == 127, -np.inf, 1.0), np.full(128, np.nan),
            np.where(np.arange(128) < 100, -0.0, 0.0), np.linspace(-7.5 * 0.75, 7.5 * 0.75, 16).repeat(8), np.full(128, -big), np.where(np.arange(128) == 9, -3.4e38, 0.0)]
    c = Case4([len(rows)], [len(rows)], kv_heads=1)
    x = torch.tensor(np.array(rows), dtype=F32, device="cuda")[:, None]
    pages, batch = c.handles(l2)
    pages.append(batch, x, x)
    back = [torch.empty_like(x) for _ in "kv"]
    pages.read(batch, *back)
    for i in range(len(rows)):
        want = quantise(x[i].cpu().numpy())
        for w in (0, 1):
            got = stored(c, w, 0, i)
            assert np.array_equal(got[1], want[1][:, 0], equal_nan=True) and np.array_equal(got[2], want[2][:, 0], equal_nan=True), (i, got[1:], want[1:])
            if np.isfinite(want[1]).all():
                assert np.array_equal(got[0], want[0]), i
                assert torch.equal(back[w][i].cpu(), values(*got, F32))
            else:
                assert back[w][i].isnan().all()


def test_sixteen_bits_are_rounded_as_the_definition_says(l2):
    """bf16 rows have many elements in the very middle of a step."""
    for io in (BF16, F16):
        c = Case4([500], [500], kv_heads=4, page=64)
        x = (torch.randn((500, 4, 128), device="cuda") * torch.rand((500, 4, 1), device="cuda") * 4).to(io)
        pages, batch = c.handles(l2)
        pages.append(batch, x, x)
        u, scale, zero = quantise(x.float().cpu().numpy())
        got = c.numbers(0, 0)
        assert np.array_equal(got[0].cpu().numpy(), u) and np.array_equal(got[1].cpu().numpy(), scale) and np.array_equal(got[2].cpu().numpy(), zero)


# ---- attention -----------------------------------------------------------------------------------------------------------

# single tokens: one position, the ends of tiles and pages, lengths with a ragged last page; a sequence without rows, one without positions
@pytest.mark.parametrize("group", [1, 3, 8, 16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("io", [F16, BF16])
def test_single_tokens(l2, io, hd, group):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 300, 555, 31]
    rows = [1] * len(kv)
    rows[-1] = 0
    compare(l2, Case4(rows, kv, hd=hd, group=group, seed=group), io)


@pytest.mark.parametrize("group", [1, 2, 5, 8, 20])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("io", [F16, BF16])
def test_chunks(l2, io, hd, group):
    compare(l2, Case4([5, 33, 64, 0, 130, 7], [5, 100, 64, 9, 150, 3], hd=hd, group=group, seed=group, page=32), io, what="small")
    compare(l2, Case4([260, 1, 300, 129], [260, 40, 731, 129], hd=hd, group=group, kv_heads=1, seed=group, layout="HND", spare_rows=3), io, what="large")
    compare(l2, Case4([2, 1, 3], [260, 700, 129], hd=hd, group=min(group, 5), seed=group), io, what="drafts")


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("hd", [64, 128])
def test_page_sizes(l2, hd, layout, page):
    for group in (4, 16):
        compare(l2, Case4([1, 1, 1], [5, 700, 257], page=page, layout=layout, group=group, hd=hd, seed=page), BF16)
    compare(l2, Case4([1, 1, 3, 70], [5, 700, 257, 290], page=page, layout=layout, group=4, hd=hd, seed=page), BF16)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (64, 4), (100, 64), (128, 17), (257, 200), (300, 256), (1000, 4), (40, 1000)])
@pytest.mark.parametrize("io", [F16, BF16])
def test_window_and_sinks(l2, io, window, sinks):
    compare(l2, Case4([1, 1, 1, 4, 1], [1, 64, 900, 300, 130], group=4, seed=window), io, window=window, sinks=sinks, what="rows")
    compare(l2, Case4([300, 140, 280], [300, 700, 290], group=2, kv_heads=1, seed=window, page=64), io, window=window, sinks=sinks, what="chunks")


def test_pages_out_of_the_window_are_not_needed(l2):
    for rows in ([1, 1], [80, 90]):
        c = Case4(rows, [1000, 777], group=2)
        q, want = run_attend(l2, c, BF16, window=200, sinks=4)
        for b in range(2):
            first = (c.kv[b] - rows[b] - 199) // 16  # the page of the first position of the first row's window
            c.table[b, 1:first] = torch.tensor([-1, 1 << 30, -(1 << 31)] * 30, dtype=torch.int32)[:first - 1]
        c.device_arrays()
        _, out = run_attend(l2, c, BF16, window=200, sinks=4, q=q)
        assert torch.equal(out, want) and int(c.status) == 0


# what a row does not see may be anything: the rest of the last page, later positions of the chunk, positions between sinks and window
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3.0e38])
@pytest.mark.parametrize("io", [F16, BF16])
def test_what_is_not_seen_does_not_matter(l2, io, value):
    def poison(c, b, j, which):
        page, off = c.slot(b, j)
        c.scales[which][page, :, off, j % 2] = value

    for rows, kv, window, sinks in (([1], [37], 0, 0), ([1], [300], 50, 3), ([6], [70], 0, 0), ([200], [333], 0, 0), ([200], [333], 60, 4), ([300], [300], 0, 0), ([40], [200], 20, 2)):
        c = Case4(rows, kv, group=2, seed=3)
        q, clean = run_attend(l2, c, io, window=window, sinks=sinks)
        used = torch.zeros((c.n_pages, c.page), dtype=torch.bool)
        for j in range(kv[0]):
            used[c.slot(0, j)] = True
        for which in (0, 1):  # every slot that holds no position
            c.scales[which].transpose(1, 2)[~used.cuda()] = value
        if window:  # positions that no row sees
            for j in range(sinks, kv[0] - rows[0] - window + 1):
                poison(c, 0, j, 0), poison(c, 0, j, 1)
        _, out = run_attend(l2, c, io, window=window, sinks=sinks, q=q)
        assert torch.equal(out, clean), (rows, kv, window)
        # a position in the middle of the chunk: rows in front of it keep their bits, rows that see it do not stay finite
        if rows[0] > 1:
            for which in (0, 1):
                j = kv[0] - rows[0] // 2
                keep = [s.clone() for s in c.scales]
                page, off = c.slot(0, j)
                c.scales[which][page, :, off] = value
                _, out = run_attend(l2, c, io, window=window, sinks=sinks, q=q)
                i = rows[0] - (kv[0] - j)
                last = min(rows[0], i + window) if window else rows[0]
                if math.isfinite(value) and which == 0 and rows[0] > 8:  # (f16 does not hold it: all rows go through bf16)
                    c.scales = keep
                    want, bound = attend4(c, q, c.hd ** -0.5, window, sinks, many=True, wide=True)
                    check(out[:i], want[:i], bound[:i]), check(out[last:], want[last:], bound[last:])
                    continue
                assert torch.equal(out[:i], clean[:i]), (rows, kv, window, which)
                if which == 1 or math.isnan(value):
                    assert not out[i:last].isfinite().any()
                assert torch.equal(out[last:], clean[last:]), (rows, kv, window, which)
                c.scales = keep


# scores that are large (the largest position decides), equal, or fall and rise along the sequence (the running maximum moves)
@pytest.mark.parametrize("io", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 150])
def test_large_and_equal_scores(l2, io, rows):
    c = Case4([rows], [500], group=2, seed=1)
    compare(l2, c, io, scale=3.0, what="large")
    compare(l2, c, io, scale=1e-6, what="equal")
    for up in (True, False):
        c = Case4([rows], [500], group=2, seed=1)
        for j in range(500):
            page, off = c.slot(0, j)
            f = 0.02 * (j if up else 499 - j) + 0.1
            c.scales[0][page, :, off] = (c.scales[0][page, :, off].float() * f * 0.05).to(BF16)
        compare(l2, c, io, scale=2.0, what="moving")


# scales of V of very different sizes side by side, in either order, at positions with much and with little weight
@pytest.mark.parametrize("io", [F16, BF16])
@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("power", [8, 20, 45])
def test_scales_of_any_size(l2, io, order, power):
    for group in (1, 8, 16):
        c = Case4([1, 1], [1500, 70], group=group, seed=2)
        for b, n in enumerate(c.kv):
            for j in range(n):
                page, off = c.slot(b, j)
                c.scales[1][page, :, off] = (c.scales[1][page, :, off].float() * 2.0 ** (order * power * (j / n - 0.5) * 2)).to(BF16)
                if j % 97 == 5:  # positions with nearly all of the weight
                    c.scales[0][page, :, off] = (c.scales[0][page, :, off].float() * 20).to(BF16)
        compare(l2, c, io, out_type=F32)  # (f16 would not hold the largest results)


def test_scale_of_zero_and_of_either_sign(l2):
    for rows in ([1], [100]):
        c = Case4(rows, [300], group=4)
        for which in (0, 1):
            c.scales[which][:, :, ::3, 0] = 0
            c.scales[which][:, :, 1::3] *= -1
        compare(l2, c, BF16)
        c.scales[1].zero_()
        _, out = run_attend(l2, c, BF16)
        assert (out == 0).all()


# the weight of a position with large V is far below the others', and the other way round: what matters is their product
@pytest.mark.parametrize("io", [F16, BF16])
@pytest.mark.parametrize("first", [True, False])
def test_a_large_value_of_little_weight(l2, io, first):
    for gap, power in ((30.0, 60), (40.0, 40), (60.0, 80)):
        c = Case4([1], [700], kv_heads=1)
        c.k.zero_()
        c.scales[0].zero_()
        page, off = c.slot(0, 3 if first else 690)
        c.scales[0][page, :, off, 1] = -gap
        c.scales[1][page, :, off] = (c.scales[1][page, :, off].float() * 2.0**power).to(BF16)
        q = torch.zeros((1, 1, 128), dtype=io, device="cuda")
        q[0, 0, 0] = 1
        compare(l2, c, io, scale=1.0, q=q, out_type=F32, what="%g %d" % (gap, power))


# queries whose elements differ in size by more than f16 holds, rows of zeros, the largest and smallest numbers of a type
@pytest.mark.parametrize("rows", [1, 60])
def test_queries_of_any_size(l2, rows):
    c = Case4([rows], [200], group=4, seed=6)
    g = torch.Generator(device="cuda").manual_seed(1)
    for io, powers in ((BF16, (-99, -30, 0, 30, 100)), (F16, (-14, 0, 15))):
        for p in powers:
            q = torch.randn((rows, c.heads, c.hd), generator=g, device="cuda") * 2.0 ** (torch.rand((rows, c.heads, c.hd), generator=g, device="cuda") * 14 - 14)
            q = (q / q.abs().amax() * 2.0**p).to(io)
            q[:, 1] = 0
            compare(l2, c, io, scale=2.0**-p if p < 100 else 2.0**-99, q=q, what="2^%d" % p)
    q = torch.randn((rows, c.heads, c.hd), device="cuda").to(BF16)
    _, clean = run_attend(l2, c, BF16, q=q)
    for value in (math.nan, math.inf):  # one row of it, and the others keep their bits
        bad = q.clone()
        bad[rows // 2, 3, 5] = value
        _, out = run_attend(l2, c, BF16, q=bad)
        assert out[rows // 2, 3].isnan().all()
        out[rows // 2, 3] = clean[rows // 2, 3]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("io", [F16, BF16])
@pytest.mark.parametrize("rows", [[1, 3], [100, 70]])
@pytest.mark.parametrize("power", [-40, -15, -9, 11, 40])
def test_values_that_f16_does_not_hold(l2, rows, io, power):
    """K and V beyond f16's range or below its normal numbers."""
    for which in (0, 1):
        c = Case4(rows, [300, 100], group=2)
        c.scales[which] = (c.scales[which].float() * 2.0**power).to(BF16)
        q = torch.randn((c.n, c.heads, c.hd), device="cuda").to(io)
        compare(l2, c, io, q=q, scale=(2.0**-power if which == 0 else 1.0) / 12, out_type=F32, what="%d" % which)
    # one position of a page that is seen, or one behind the last of a sequence
    c = Case4(rows, [300, 100], group=2)
    page, off = c.slot(0, 250)
    c.scales[1][page, :, off] = (c.scales[1][page, :, off].float() * 2.0**power).to(BF16)
    page, off = int(c.table[1, 6]), 15
    c.scales[0][page, :, off], c.scales[1][page, :, off] = 1e30, -1e30
    compare(l2, c, io, out_type=F32, what="one")


def test_output_in_32_bits_and_strides(l2):
    for io in (F16, BF16):
        c = Case4([1, 90, 3], [200, 400, 3], group=2, seed=9)
        compare(l2, c, io, out_type=F32, what="f32")
        big = torch.randn((c.n, 2, c.heads + 4, c.hd), device="cuda").to(io)
        q = big[:, 1, 2:2 + c.heads]
        room = torch.full((c.heads, c.n, c.hd + 8), 3.0, dtype=io, device="cuda")
        out = room[:, :, :c.hd].transpose(0, 1)
        pages, batch = c.handles(l2)
        pages.attend(batch, q, out)
        _, plain = run_attend(l2, c, io, q=q.contiguous())
        assert torch.equal(out, plain) and (room[:, :, c.hd:] == 3.0).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_pool_with_gaps(l2, hd):
    """Strides that are no multiples of one another: 16 bytes behind every head, 48 behind every position, 80 behind every page."""
    for rows, kv in (([1, 1], [100, 37]), ([70, 200], [150, 260])):
        a = Case4(rows, kv, group=2, hd=hd, seed=11)
        q, want = run_attend(l2, a, BF16)
        head, pos = hd // 2 + 16, 2 * (hd // 2 + 16) + 48
        page = a.page * pos + 80
        pools = []
        for t in (a.k, a.v):
            flat = torch.zeros(a.n_pages * page + hd, dtype=torch.uint8, device="cuda")
            view = flat.as_strided((a.n_pages, a.page, 2, hd // 2), (page, pos, head, 1))
            view.copy_(t)
            pools.append(view)
        a.k, a.v = pools
        _, out = run_attend(l2, a, BF16, q=q)
        assert torch.equal(out, want)
        new = torch.randn((a.n, 2, hd), device="cuda")
        back = [torch.zeros_like(new) for _ in "kv"]
        pages, batch = a.handles(l2)
        pages.append(batch, new, new)
        pages.read(batch, *back)
        u, scale, zero = quantise(new.cpu().numpy())
        assert torch.equal(back[0], back[1]) and torch.equal(back[0].cpu(), values(u, scale[..., 0], zero[..., 0], F32))


def test_more_rows_than_positions(l2):
    """Rows of negative positions see nothing: 0, whole blocks of them too."""
    for rows, kv in (([600, 1, 3], [5, 0, 0]), ([300], [0]), ([9, 1], [4, 2]), ([3, 1], [1, 0])):
        c = Case4(rows, kv, group=2, seed=2)
        compare(l2, c, BF16)
        compare(l2, c, F16, window=3, sinks=1)


def test_offsets_beyond_32_bits(l2):
    """Pages whose elements, and bytes, start beyond 2^32."""
    n_pages = (5 << 30) // (256 * 2 * 64)
    for layout in ("NHD", "HND"):
        c = Case4([1, 70], [300, 200], page=256, n_pages=n_pages, layout=layout)
        top = torch.tensor([n_pages - 1, n_pages - 2, n_pages - 5], dtype=torch.int32)
        c.table[0, :2], c.table[1, :1] = top[:2], top[2:]
        c.device_arrays()
        compare(l2, c, BF16)
        back = [torch.zeros((c.n, 2, 128), dtype=F32, device="cuda") for _ in "kv"]
        pages, batch = c.handles(l2)
        new = torch.randn((c.n, 2, 128), device="cuda")
        pages.append(batch, new, new)
        pages.read(batch, *back)
        u, scale, zero = quantise(new.cpu().numpy())
        assert torch.equal(back[0], back[1]) and torch.equal(back[0].cpu(), values(u, scale[..., 0], zero[..., 0], F32))
        del c, pages


def test_many_sequences_and_splits(l2):
    """More sequences than a CTA has threads, some without rows; one long sequence among short ones, so that its positions are split."""
    n = 1111
    rng = np.random.default_rng(0)
    kv = rng.integers(0, 40, n).tolist()
    compare(l2, Case4([int(x > 5) for x in kv], kv, group=1, hd=64, page=8, kv_heads=1), BF16)
    rows, kv = [1] * 20, rng.integers(1, 60, 20).tolist()
    kv[7] = 30000
    compare(l2, Case4(rows, kv, group=8), BF16)
    compare(l2, Case4([40, 3], [20000, 3], group=8, kv_heads=1), BF16)


@pytest.mark.parametrize("tokens,group", [(1, 1), (1, 3), (3, 3), (2, 8), (2, 20)])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_pieces(l2, hd, tokens, group):
    compare(l2, Case4([tokens], [25001], hd=hd, group=group, kv_heads=1, page=64), BF16)


def test_single_tokens_among_chunks(l2):
    """Both kernels in one call: a single token's result is that of the kernel for few rows."""
    c = Case4([1, 120, 1, 40, 1], [300, 400, 7, 900, 1000], group=4, seed=8)
    q, out = run_attend(l2, c, F16, out_type=F32)
    want, bound = attend4(c, q, c.hd ** -0.5)
    more = attend4(c, q, c.hd ** -0.5, many=True)[1]
    single = torch.tensor([n == 1 for n in c.rows for _ in range(n)], device="cuda")
    check(out, want, torch.where(single[:, None, None], bound, more))


def test_same_bits_every_time(l2):
    for rows, kv in (([1] * 9, [700, 3, 5000, 64, 1, 90, 1200, 333, 2]), ([300, 200], [3000, 200])):
        c = Case4(rows, kv, group=4)
        q, first = run_attend(l2, c, BF16)
        for _ in range(3):
            assert torch.equal(run_attend(l2, c, BF16, q=q)[1], first)


def test_many_small_probabilities(l2):
    """One position with most of the weight and very many with little: together the little ones matter."""
    for io in (F16, BF16):
        c = Case4([1], [20000], kv_heads=1, seed=4)
        c.k.zero_(), c.v.fill_(0xff)
        c.scales[0].zero_()
        c.scales[1][..., 0], c.scales[1][..., 1] = 0.0625, 0
        page, off = c.slot(0, 7)
        c.scales[0][page, :, off, 1] = 11
        c.v[page, off] = 0
        q = torch.zeros((1, 1, 128), dtype=io, device="cuda")
        q[0, 0, 0] = 1
        compare(l2, c, io, scale=1.0, q=q)


def test_bad_pages_and_lengths_are_reported(l2):
    c = Case4([1, 70], [100, 150], group=2)
    q, clean = run_attend(l2, c, BF16)
    c.table[0, 3], c.table[1, 5] = c.n_pages, -7
    c.device_arrays()
    _, out = run_attend(l2, c, BF16, q=q)
    assert int(c.status) == l2.paged.BAD_PAGE and out.isfinite().all()
    new = torch.randn((c.n, 2, 128), device="cuda")
    before = c.k.clone()
    c.table[1, 5:] = -7
    c.device_arrays()
    pages, batch = c.handles(l2)
    pages.append(batch, new, new)
    back = [torch.full_like(new, 7.0) for _ in "kv"]
    pages.read(batch, *back)
    assert int(c.status) == l2.paged.BAD_PAGE
    for i in range(70):
        assert bool((back[0][1 + i] == 0).all()) == (80 + i >= 80)  # all of them lie in pages that are none: read as zeros
    assert torch.equal(c.k[c.table[1, :5].long().cuda()], before[c.table[1, :5].long().cuda()])


def test_in_a_graph(l2):
    """A step captured once and replayed with other lengths and rows."""
    for rows in ([1, 1, 1], [40, 1, 90]):
        c = Case4(rows, [300, 20, 500], group=4)
        new = torch.randn((c.n, 2, 128), device="cuda")
        q = torch.randn((c.n, c.heads, 128), device="cuda").to(BF16)
        out = torch.zeros_like(q)
        pages, batch = c.handles(l2)
        work = torch.empty(pages.workspace_bytes(batch, c.heads), dtype=torch.uint8, device="cuda")
        step = lambda: (pages.append(batch, new, new), pages.attend(batch, q, out, workspace=work))  # noqa: E731
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for kv in ([300, 20, 500], [250, 1, 499], [40, 17, 90]):
            c.kv = kv
            c.d_kv.copy_(torch.tensor(kv, dtype=torch.int32))
            new.normal_(), q.normal_()
            graph.replay()
            torch.cuda.synchronize()
            want, bound = attend4(c, q, 128 ** -0.5, many=rows[0] > 1)
            check(out, want, bound)
            assert int(c.status) == 0

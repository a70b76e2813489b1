"""The paged KV cache (append, read back) and its attention against the same in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged_reference import Case, attend, check  # noqa: E402

F16, BF16, I8, F32 = torch.float16, torch.bfloat16, torch.int8, torch.float32
CACHES = [(F16, F16), (BF16, BF16), (I8, BF16), (I8, F16)]  # cache, queries


def p_unit(cache, q):
    """The probabilities are rounded to q's type, with an int8 cache to bf16 (and the scale product is rounded in f32 first)."""
    return None if cache != I8 else 2.0**-8 * (1 + 2.0**-10)


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
    cache = c.k.dtype
    want, bound = attend(c, q, scale or c.hd ** -0.5, window, sinks, p_unit(cache, io))
    n = int(c.row_start[-1])
    check(out[:n], want[:n], bound[:n], what)
    assert (out[n:] == 7.0).all()  # rows of no sequence are left alone
    assert int(c.status) == 0


# ---- attention ---------------------------------------------------------------------------------------------------------

# single tokens: one position, the ends of tiles and pages, lengths with a ragged last page; a sequence without rows, one without positions
@pytest.mark.parametrize("group", [1, 3, 8, 16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cache,io", CACHES)
def test_single_tokens(l2, cache, io, hd, group):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 300, 555, 31]
    rows = [1] * len(kv)
    rows[-1] = 0
    compare(l2, Case(rows, kv, hd=hd, group=group, cache=cache, seed=group), io)


# chunks: fewer and more rows than a tile has, whole prompts, chunks behind a context, more rows than positions
@pytest.mark.parametrize("group", [1, 2, 5, 8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cache,io", CACHES)
def test_chunks(l2, cache, io, hd, group):
    compare(l2, Case([5, 33, 64, 0, 130, 7], [5, 100, 64, 9, 150, 3], hd=hd, group=group, cache=cache, seed=group, page=32), io, what="small")
    compare(l2, Case([260, 1, 300, 129], [260, 40, 731, 129], hd=hd, group=group, kv_heads=1, cache=cache, seed=group, layout="HND", spare_rows=3), io, what="large")


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("cache,io", [CACHES[1], CACHES[2]])
def test_page_sizes(l2, cache, io, layout, page):
    compare(l2, Case([1, 1, 3, 70], [5, 700, 257, 290], page=page, layout=layout, cache=cache, group=4, seed=page), io)


# windows smaller and larger than a tile, sinks that end inside a tile, overlap the window or lie in front of it
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (64, 4), (100, 64), (128, 17), (257, 200), (1000, 4), (40, 1000)])
@pytest.mark.parametrize("cache,io", [CACHES[0], CACHES[2]])
def test_window_and_sinks(l2, cache, io, window, sinks):
    compare(l2, Case([1, 1, 1, 6, 1], [1, 64, 900, 300, 130], cache=cache, group=4, seed=window), io, window=window, sinks=sinks, what="rows")
    compare(l2, Case([300, 140, 280], [300, 700, 290], cache=cache, group=2, kv_heads=1, seed=window, page=64), io, window=window, sinks=sinks, what="chunks")


@pytest.mark.parametrize("cache,io", [CACHES[1], CACHES[2]])
def test_pages_out_of_the_window_are_not_needed(l2, cache, io):
    for rows in ([1, 1], [80, 90]):
        c = Case(rows, [1000, 777], cache=cache, group=2)
        q, want = run_attend(l2, c, io, window=200, sinks=4)
        for b in range(2):
            first = (c.kv[b] - rows[b] - 199) // 16  # the page of the first position of the first row's window
            c.table[b, 1:first] = torch.tensor([-1, 1 << 30, -(1 << 31)] * 30, dtype=torch.int32)[:first - 1]
        c.device_arrays()
        _, out = run_attend(l2, c, io, window=200, sinks=4, q=q)
        assert torch.equal(out, want) and int(c.status) == 0


def poison(c, b, j, value, which):
    t = (c.k, c.v)[which]
    page, off = c.slot(b, j)
    if t.dtype == I8:
        c.scales[which][page, :, off] = value
    elif c.layout == "NHD":
        t[page, off, :, ::3] = value
    else:
        t[page, :, off, ::3] = value


# what a row does not see may be anything: the rest of the last page, later positions of the chunk, positions between sinks and window
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cache,io", CACHES)
def test_what_is_not_seen_does_not_matter(l2, cache, io, value):
    for rows, kv, window, sinks in (([1], [37], 0, 0), ([1], [300], 50, 3), ([6], [70], 0, 0), ([200], [333], 0, 0), ([200], [333], 60, 4), ([300], [300], 0, 0), ([40], [200], 20, 2)):
        c = Case(rows, kv, cache=cache, group=2, seed=3)
        q, clean = run_attend(l2, c, io, window=window, sinks=sinks)
        used = {c.slot(0, j) for j in range(kv[0])}
        for page in range(c.n_pages):  # every slot that holds no position
            for off in range(c.page):
                if (page, off) not in used:
                    for which in (0, 1):
                        c.table[0, -1] = page  # (the last entry of the table belongs to no position)
                        poison(c, 0, (c.table.shape[1] - 1) * c.page + off, value, which)
        if window:  # positions that no row sees
            for j in range(sinks, kv[0] - rows[0] - window + 1):
                poison(c, 0, j, value, 0), poison(c, 0, j, value, 1)
        _, out = run_attend(l2, c, io, window=window, sinks=sinks, q=q)
        assert torch.equal(out, clean), (rows, kv, window)
        # a position in the middle of the chunk: rows in front of it keep their bits, rows that see it do not stay finite
        if rows[0] > 1:
            for which in (0, 1):
                j = kv[0] - rows[0] // 2
                keep = (c.k.clone(), c.v.clone(), [None if s is None else s.clone() for s in c.scales])
                poison(c, 0, j, value, which)
                _, out = run_attend(l2, c, io, window=window, sinks=sinks, q=q)
                i = rows[0] - (kv[0] - j)
                assert torch.equal(out[:i], clean[:i]), (rows, kv, window, which)
                last = min(rows[0], i + window) if window else rows[0]
                seen = out[i:last]
                if which == 1:
                    hit = seen if cache == I8 else seen[..., ::3]
                    assert not hit.isfinite().any()
                elif math.isnan(value):
                    assert seen.isnan().all()
                assert torch.equal(out[last:], clean[last:]), (rows, kv, window, which)
                c.k, c.v, c.scales = keep


# scores that are large (the largest position decides), equal, or fall and rise along the sequence (the running maximum moves)
@pytest.mark.parametrize("cache,io", CACHES)
@pytest.mark.parametrize("rows", [1, 150])
def test_large_and_equal_scores(l2, cache, io, rows):
    c = Case([rows], [500], cache=cache, group=2, seed=1)
    compare(l2, c, io, scale=30.0, what="large")
    compare(l2, c, io, scale=1e-6, what="equal")
    for up in (True, False):
        c = Case([rows], [500], cache=cache, group=2, seed=1)
        for j in range(500):
            page, off = c.slot(0, j)
            f = 0.02 * (j if up else 499 - j) + 0.1
            if cache == I8:
                c.scales[0][page, :, off] = 0.003 * f
            else:
                c.k[page, off] *= f
        compare(l2, c, io, scale=2.0, what="moving")


def test_output_in_32_bits_and_strides(l2):
    for cache, io in CACHES:
        c = Case([1, 90, 3], [200, 400, 3], cache=cache, group=2, seed=9)
        compare(l2, c, io, out_type=F32, what="f32")
        # queries that are a part of a fused projection's rows, heads in another order, an output with a gap between its rows
        big = torch.randn((c.n, 2, c.heads + 4, c.hd), device="cuda").to(io)
        q = big[:, 1, 2:2 + c.heads]
        room = torch.full((c.heads, c.n, c.hd + 8), 3.0, dtype=io, device="cuda")
        out = room[:, :, :c.hd].transpose(0, 1)
        pages, batch = c.handles(l2)
        pages.attend(batch, q, out)
        _, plain = run_attend(l2, c, io, q=q.contiguous())
        assert torch.equal(out, plain) and (room[:, :, c.hd:] == 3.0).all()


def test_pool_with_strides(l2):
    """K and V side by side in one allocation of several layers."""
    for cache, io in (CACHES[0], CACHES[2]):
        a = Case([1, 70], [100, 150], cache=cache, group=2)
        pool = torch.zeros((a.n_pages, 3, 2, a.page, a.kv_heads, a.hd), dtype=cache, device="cuda")
        pool[:, 1, 0], pool[:, 1, 1] = a.k, a.v
        q, want = run_attend(l2, a, io)
        a.k, a.v = pool[:, 1, 0], pool[:, 1, 1]
        _, out = run_attend(l2, a, io, q=q)
        assert torch.equal(out, want)


@pytest.mark.parametrize("cache,io", CACHES)
@pytest.mark.parametrize("hd", [64, 128])
def test_pool_with_gaps(l2, cache, io, hd):
    """Strides that are no multiples of one another: a gap of 16 bytes behind every head, another behind every position, another behind every page."""
    gap = 16 if cache == I8 else 8
    for rows, kv in (([1, 1], [100, 37]), ([70, 200], [150, 260])):
        a = Case(rows, kv, cache=cache, group=2, hd=hd, seed=11)
        q, want = run_attend(l2, a, io)
        head, pos = hd + gap, 2 * (hd + gap) + 3 * gap
        page = a.page * pos + 5 * gap
        pools = []
        for t in (a.k, a.v):
            flat = torch.zeros(a.n_pages * page + hd, dtype=cache, device="cuda")
            view = flat.as_strided((a.n_pages, a.page, 2, hd), (page, pos, head, 1))
            view.copy_(t)
            pools.append(view)
        a.k, a.v = pools
        _, out = run_attend(l2, a, io, q=q)
        assert torch.equal(out, want)
        new = torch.randn((a.n, 2, hd), device="cuda").to(io)
        back = [torch.zeros_like(new) for _ in "kv"]
        pages, batch = a.handles(l2)
        pages.append(batch, new, new)
        pages.read(batch, *back)
        assert torch.equal(back[0], back[1]) and (cache == I8 or torch.equal(back[0], new))


@pytest.mark.parametrize("cache,io", CACHES)
def test_more_rows_than_positions(l2, cache, io):
    """Rows of negative positions see nothing: 0, whole blocks of them too."""
    for rows, kv in (([600, 1, 3], [5, 0, 0]), ([300], [0]), ([9, 1], [4, 2])):
        c = Case(rows, kv, cache=cache, group=2, seed=2)
        compare(l2, c, io)
        compare(l2, c, io, window=3, sinks=1)


@pytest.mark.parametrize("cache,io", [CACHES[1], CACHES[2]])
def test_offsets_beyond_32_bits(l2, cache, io):
    """Pages whose elements, and bytes, start beyond 2^32."""
    n_pages = (5 << 30) // (256 * 2 * 128 * (1 if cache == I8 else 2)) * (1 if cache == I8 else 2)
    for layout in ("NHD", "HND"):
        c = Case([1, 70], [300, 200], cache=cache, page=256, n_pages=n_pages, layout=layout)
        top = torch.tensor([n_pages - 1, n_pages - 2, n_pages - 5], dtype=torch.int32)
        c.table[0, :2], c.table[1, :1] = top[:2], top[2:]
        c.device_arrays()
        compare(l2, c, io)
        back = [torch.zeros((c.n, 2, 128), dtype=F32, device="cuda") for _ in "kv"]
        pages, batch = c.handles(l2)
        new = torch.randn((c.n, 2, 128), device="cuda").to(io)
        pages.append(batch, new, new)
        pages.read(batch, *back)
        tol = 0.51 * new.abs().amax(-1, keepdim=True).float() / 127 if cache == I8 else 0.0
        assert ((back[0] - new.float()).abs() <= tol).all() and torch.equal(back[0], back[1])
        del c, pages


def test_many_sequences_and_splits(l2):
    """More sequences than a CTA has threads, some without rows; one long sequence among short ones, so that its positions are split."""
    n = 1111
    rng = np.random.default_rng(0)
    kv = rng.integers(0, 40, n).tolist()
    rows = [int(x > 5) for x in kv]
    compare(l2, Case(rows, kv, group=1, hd=64, cache=BF16, page=8, kv_heads=1), BF16)
    rows, kv = [1] * 20, rng.integers(1, 60, 20).tolist()
    kv[7] = 30000
    compare(l2, Case(rows, kv, group=8, cache=I8), BF16)
    compare(l2, Case([40, 3], [20000, 3], group=8, kv_heads=1, cache=BF16), BF16)


# one pair cut into more pieces than a warp has threads: few rows (1, 3, 9, 16) and a block of 2 x 20
@pytest.mark.parametrize("tokens,group", [(1, 1), (1, 3), (3, 3), (2, 8), (2, 20)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cache,io", [CACHES[1], CACHES[3]])
def test_many_pieces(l2, cache, io, hd, tokens, group):
    compare(l2, Case([tokens], [25001], hd=hd, group=group, cache=cache, kv_heads=1, page=64), io)


def test_same_bits_every_time(l2):
    for rows, kv in (([1] * 9, [700, 3, 5000, 64, 1, 90, 1200, 333, 2]), ([300, 200], [3000, 200])):
        c = Case(rows, kv, cache=BF16, group=4)
        q, first = run_attend(l2, c, BF16)
        for _ in range(3):
            assert torch.equal(run_attend(l2, c, BF16, q=q)[1], first)


def test_sums_do_not_depend_on_small_probabilities_being_lost(l2):
    """One position with most of the weight and very many with little: together the little ones matter (f16 would lose them as they are)."""
    for cache, io in CACHES:
        c = Case([1], [20000], kv_heads=1, cache=cache, seed=4)
        c.k.fill_(0), c.v.fill_(1)
        if cache == I8:
            c.scales[0].fill_(1.0), c.scales[1].fill_(0.01)
        page, off = c.slot(0, 7)
        c.k[page, off, 0, 0] = 11
        c.v[page, off] = 0
        q = torch.zeros((1, 1, 128), dtype=io, device="cuda")
        q[0, 0, 0] = 1
        compare(l2, c, io, scale=1.0, q=q)


# ---- append and read ------------------------------------------------------------------------------------------------------

def rotate(x, cos, sin, pos):
    h = x.shape[-1] // 2
    a, b = x[..., :h].double(), x[..., h:].double()
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("cache", [F16, BF16, I8])
def test_append_and_read(l2, cache, io, layout, hd, rope):
    for rows, kv in (([1, 1, 0, 1], [1, 33, 5, 64]), ([70, 1, 300, 5], [90, 7, 300, 3]), ([1], [1])):
        c = Case(rows, kv, kv_heads=3, hd=hd, cache=cache, layout=layout, spare_rows=2)
        g = torch.Generator(device="cuda").manual_seed(3)
        k, v = (torch.randn((c.n, 3, hd), generator=g, device="cuda").to(io) for _ in "kv")
        q = torch.randn((c.n, 6, hd), generator=g, device="cuda").to(io)
        q_out = torch.full((c.n, 6, hd), 7.0, dtype=BF16, device="cuda")
        before = c.k.clone(), c.v.clone(), [None if s is None else s.clone() for s in c.scales]
        angle = torch.rand((400, hd // 2), generator=g, device="cuda") * 6
        cos, sin = angle.cos(), angle.sin()
        pages, batch = c.handles(l2)
        pages.append(batch, k, v, rope=(cos, sin) if rope else None, q=q, q_out=q_out)
        back = [torch.full((c.n, 3, hd), 7.0, dtype=F32, device="cuda") for _ in "kv"]
        pages.read(batch, *back)
        torch.cuda.synchronize()
        assert int(c.status) == 0
        touched = torch.zeros((c.n_pages, c.page), dtype=torch.bool)
        for b in range(len(rows)):
            for i in range(rows[b]):
                r, p = int(c.row_start[b]) + i, kv[b] - rows[b] + i
                if p < 0:  # more rows than positions: nothing is written
                    assert (back[0][r] == 7.0).all() and (q_out[r] == 7.0).all()
                    continue
                touched[c.slot(b, p)] = True
                want = [x[r:r + 1].double() for x in (k, v, q)]
                if rope:
                    want[0], want[2] = (rotate(x[r:r + 1], cos, sin, torch.tensor([p])) for x in (k, q))
                # three roundings of the rotation in f32, of products of up to |x|
                turn = 3 * 2.0**-24 * max(float(w.abs().max()) for w in want) * 2
                check(q_out[r:r + 1], want[2], torch.full_like(want[2], turn if rope else 0.0), "q")
                for which in (0, 1):
                    w = want[which][0]
                    got = back[which][r].double()
                    if cache == I8:
                        step = w.abs().amax(-1, keepdim=True) / 127
                        room = step * (0.5 + 127 * 2.0**-21) + turn
                    else:
                        room = w.abs() * (2.0**-11 if cache == F16 else 2.0**-8) + 2.0**-24 + turn
                    assert ((got - w).abs() <= room).all()
        assert (back[0][int(c.row_start[-1]):] == 7.0).all()
        # nothing else has been written
        for new, old in zip((c.k, c.v), before):
            a, o = (t if layout == "NHD" else t.transpose(1, 2) for t in (new, old if not isinstance(old, list) else None))
            assert torch.equal(a.cpu()[~touched], o.cpu()[~touched])
        for new, old in zip(c.scales, before[2]):
            if new is not None:
                assert torch.equal(new.transpose(1, 2).cpu()[~touched], old.transpose(1, 2).cpu()[~touched])


@pytest.mark.parametrize("hd", [64, 128])
def test_int8_rows_that_are_special(l2, hd):
    c = Case([8], [8], kv_heads=1, hd=hd, cache=I8)
    x = torch.randn((8, 1, hd), device="cuda")
    x[1] = 0
    x[2] = 1e-35 * x[2]       # below what is resolved
    x[3, 0, 5] = math.nan
    x[4, 0, hd - 1] = -math.inf
    x[5] = torch.finfo(F32).max * torch.sign(x[5])
    x[6] = 2.0**-99 * torch.sign(x[6])
    x[7] = -127 * torch.sign(x[7])
    x[7, 0, 1:] = (torch.arange(hd - 1, device="cuda") % 250 - 124) + 0.5  # ties go to even
    pages, batch = c.handles(l2)
    back = [torch.zeros((8, 1, hd), device="cuda") for _ in "kv"]
    pages.append(batch, x, x)
    pages.read(batch, *back)
    assert torch.equal(back[0].nan_to_num(9), back[1].nan_to_num(9))
    got = back[0]
    assert (got[1] == 0).all() and (got[2] == 0).all() and got[3].isnan().all() and got[4].isnan().all()
    for i in (0, 5, 6):
        step = x[i].abs().max().double() / 127
        assert ((got[i].double() - x[i].double()).abs() <= step * 0.501).all()
    page, off = c.slot(0, 7)
    assert torch.equal(c.k[page, off, 0, 1:].float(), torch.round(x[7, 0, 1:]))


def test_strided_rows(l2):
    c = Case([40, 1], [50, 9], kv_heads=2, cache=BF16)
    qkv = torch.randn((c.n, 4 + 2 + 2, 128), device="cuda").to(BF16)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    q_out = torch.empty((4, c.n, 128), dtype=BF16, device="cuda").transpose(0, 1)
    pages, batch = c.handles(l2)
    pages.append(batch, k, v, q=q, q_out=q_out)
    k_back = torch.empty((2, c.n, 128), dtype=BF16, device="cuda").transpose(0, 1)
    v_back = torch.empty((c.n, 2, 256), dtype=BF16, device="cuda")[..., :128]
    pages.read(batch, k_back, v_back)
    assert torch.equal(k_back, k) and torch.equal(v_back, v) and torch.equal(q_out, q)


# ---- what only the device can see -------------------------------------------------------------------------------------------

def test_status_bits(l2):
    from llama2_rs import paged
    for cache, io in (CACHES[1], CACHES[2]):
        for rows, kv in (([1, 1, 1], [40, 50, 60]), ([100, 90, 120], [140, 150, 160])):
            def fresh():
                return Case(rows, kv, cache=cache, group=2)

            c = fresh()
            q, clean = run_attend(l2, c, io)
            last = int(c.row_start[2])
            for bad in (-1, c.n_pages, 1 << 30):  # a page that is needed: only its sequence changes, and stays finite
                c = fresh()
                c.d_table[1, 1] = bad
                _, out = run_attend(l2, c, io, q=q)
                assert int(c.status) == paged.BAD_PAGE and out.isfinite().all()
                assert torch.equal(out[:rows[0]], clean[:rows[0]]) and torch.equal(out[last:], clean[last:])
            c = fresh()
            c.d_kv[1] = 1 << 29
            _, out = run_attend(l2, c, io, q=q)
            assert int(c.status) & paged.BAD_LENGTH and torch.equal(out[last:], clean[last:])
            c = fresh()
            c.d_kv[1] = -4
            _, out = run_attend(l2, c, io, q=q)
            assert int(c.status) == paged.BAD_LENGTH and (out[rows[0]:last] == 0).all()
            c = fresh()
            c.d_start[2] = c.n + 5
            _, out = run_attend(l2, c, io, q=q)
            assert int(c.status) & paged.BAD_ROWS and torch.equal(out[:rows[0]], clean[:rows[0]])
            c = fresh()  # more rows than max_rows says
            _, out = run_attend(l2, c, io, q=q, max_rows=max(rows) - 1 if rows[0] > 1 else None)
            assert (int(c.status) == paged.BAD_ROWS) == (rows[0] > 1)
    c = Case([1, 1], [40, 50], cache=F16)
    pages, batch = c.handles(l2)
    k = torch.randn((2, 2, 128), device="cuda")
    cos = torch.ones((45, 64), device="cuda")
    old = c.k.clone()
    pages.append(batch, k, k, rope=(cos, cos * 0))
    assert int(c.status) == paged.BAD_ROPE
    page, off = c.slot(1, 49)
    assert torch.equal(c.k[page, off], old[page, off])
    page, off = c.slot(0, 39)
    assert torch.equal(c.k[page, off], k[0].half())


# ---- streams, graphs, workspaces ---------------------------------------------------------------------------------------------

def test_streams_and_graph(l2):
    c = Case([1, 1, 90], [600, 3000, 400], cache=BF16, group=4)
    q, want = run_attend(l2, c, BF16)
    pages, batch = c.handles(l2)
    work = torch.empty(pages.workspace_bytes(batch, c.heads), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    out = torch.zeros_like(q)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pages.attend(batch, q, out, workspace=work)
    s.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    torch.cuda.synchronize()
    pages.attend(batch, q, out, workspace=work, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.append(batch, q[:, :2], q[:, 2:4])
        pages.attend(batch, q, out, workspace=work)
    pages.append(batch, q[:, :2], q[:, 2:4])
    _, want = run_attend(l2, c, BF16, q=q)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    work.fill_(255)  # whatever the workspace holds
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals_of_the_python_objects(l2):
    c = Case([1, 2], [5, 6], cache=F16)
    pages, batch = c.handles(l2)
    q = torch.zeros((3, 2, 128), dtype=F16, device="cuda")
    for bad in (lambda: l2.KvPages(c.k, c.v.float()), lambda: l2.KvPages(c.k, c.v, torch.zeros(1), torch.zeros(1)), lambda: l2.KvPages(c.k.cpu(), c.v.cpu()),
                lambda: l2.KvPages(c.k.to(I8), c.v.to(I8)), lambda: l2.KvPages(c.k, c.v, layout="XYZ"),
                lambda: l2.KvBatch(c.d_table.long(), c.d_kv, c.d_start, 3, 2), lambda: l2.KvBatch(c.d_table, c.d_kv, c.d_kv, 3, 2),
                lambda: pages.attend(batch, q[:2], q), lambda: pages.attend(batch, q, q[:, :1]), lambda: pages.attend(batch, q.cpu(), q),
                lambda: pages.attend(batch, q, q, stream=0), lambda: pages.append(batch, q, q, q=q), lambda: pages.append(batch, q[:, :1], q)):
        with pytest.raises((ValueError, l2.L2Error)):
            bad()
    for bad in (lambda: pages.attend(batch, q.bfloat16(), q.bfloat16()), lambda: pages.attend(batch, q.float(), q), lambda: pages.attend(batch, q, q.bfloat16()),
                lambda: pages.attend(batch, q, q, window=-1), lambda: pages.attend(batch, q, q, scale=math.nan), lambda: pages.attend(batch, q, q, scale=0.0),
                lambda: pages.attend(batch, q, q, workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(l2.L2Error) as e:
            bad()
        assert e.value.code == -1
    empty = Case([0, 0], [5, 6], cache=F16)
    none = torch.zeros((0, 2, 128), dtype=F16, device="cuda")
    pages, batch = empty.handles(l2)
    pages.attend(batch, none, none)
    pages.append(batch, none, none)
    pages.read(batch, none, none)


# the workspace may hold anything, whatever the cuts of the work are: few and many sequences, pieces of one sequence, singles among chunks
@pytest.mark.parametrize("cache,io", [CACHES[1], CACHES[2]])
@pytest.mark.parametrize("rows,kv,group", [([1], [5000], 1), ([1] * 24, list(range(30, 2500, 103)), 1), ([1] * 40, [7] * 39 + [9000], 4), ([5] * 12, list(range(300, 3000, 225)), 8),
                                           ([300, 1, 290, 1, 1], [2000, 1500, 300, 40, 3000], 2), ([700], [700], 1)])
def test_workspace_contents_do_not_matter(l2, cache, io, rows, kv, group):
    c = Case(rows, kv, kv_heads=8, group=group, cache=cache)
    q, want = run_attend(l2, c, io)
    pages, batch = c.handles(l2)
    work = torch.empty(pages.workspace_bytes(batch, c.heads), dtype=torch.uint8, device="cuda")
    for fill in (0, 1, 127, 255):
        work.fill_(fill)
        out = torch.full_like(q, 7.0)
        pages.attend(batch, q, out, workspace=work)
        assert torch.equal(out, want), fill
    assert int(c.status) == 0

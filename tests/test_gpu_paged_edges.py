"""The paged cache and its attention at the edges of what they are given."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged_reference import Case  # noqa: E402
from test_gpu_paged import BF16, CACHES, F16, I8, compare, run_attend  # noqa: E402


# a large element of q where K has nothing stored: the others count as much as without it (up to 8 rows, up to 16, a block of rows)
@pytest.mark.parametrize("tokens,group", [(1, 1), (1, 8), (2, 4), (1, 16), (3, 5), (40, 2)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cache,io,large", [(I8, BF16, 1e4), (I8, BF16, 1e6), (I8, BF16, 1e30), (I8, F16, 6e4), (BF16, BF16, 1e30), (F16, F16, 6e4)])
def test_elements_of_q_that_are_far_apart(l2, cache, io, large, hd, tokens, group):
    c = Case([tokens], [512], group=group, hd=hd, cache=cache, seed=6)
    c.k[..., 5] = 0
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.randn((c.n, c.heads, hd), generator=g, device="cuda")
    q[..., 5] = large
    compare(l2, c, io, q=q.to(io), what="large %g" % large)


# a table that is too short for the length a step states: nothing is written over what the table does hold, nothing is read from the wrong place
@pytest.mark.parametrize("length", [65, 66, 1 << 29, (1 << 31) - 1, -1, -(1 << 31)])
@pytest.mark.parametrize("cache,io", CACHES)
def test_append_and_read_leave_out_a_length_beyond_the_table(l2, cache, io, length):
    from llama2_rs import paged
    c = Case([1, 3, 2], [40, 64, 60], cache=cache, page=16)
    c.table = c.table[:, :4].contiguous()
    c.device_arrays()
    c.d_kv[1] = length
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((c.n, 2, 128), generator=g, device="cuda").to(io) for _ in "kv")
    q_out = torch.full((c.n, 2, 128), 7.0, dtype=io, device="cuda")
    back = [torch.full((c.n, 2, 128), 7.0, device="cuda") for _ in "kv"]
    before = [None if t is None else t.clone() for t in (c.k, c.v, *c.scales)]
    pages, batch = c.handles(l2)
    pages.append(batch, k, v, q=k, q_out=q_out)
    assert int(c.status) == paged.BAD_LENGTH
    mine = [c.slot(1, j) for j in range(64)]
    for new, old in zip((c.k, c.v, *c.scales), before):
        if new is not None:
            for page, off in mine:
                assert torch.equal(c.at(new, page, off), c.at(old, page, off)), (page, off)
    assert (q_out[1:4] == 7.0).all() and torch.equal(q_out[:1], k[:1]) and torch.equal(q_out[4:], k[4:])
    c.status.zero_()
    pages.read(batch, *back)
    assert int(c.status) == paged.BAD_LENGTH
    for t, new in zip(back, (k, v)):
        assert (t[1:4] == 7.0).all()
        for r in (0, 4, 5):  # the others are there
            step = new[r].float().abs().amax(-1, keepdim=True) / 127 if cache == I8 else 0.0
            assert ((t[r] - new[r].float()).abs() <= 0.51 * step).all()


# a position that a row sees, whose probability is too small for any number, holds a NaN or an infinity: 0 x NaN is NaN wherever the row lies in a tile
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("tokens,group,window", [(1, 2, 0), (100, 2, 0), (100, 2, 90), (8, 16, 70), (60, 1, 0)])
@pytest.mark.parametrize("io", [F16, BF16])
def test_a_scale_that_is_not_finite_behind_a_probability_of_zero(l2, io, tokens, group, window, value):
    c = Case([tokens], [200], cache=I8, group=group, seed=8)
    c.k.clamp_(1, 2)  # (with queries of ones no score is far below the others)
    j = 160 if tokens > 40 else 199 - tokens // 2
    page, off = c.slot(0, j)
    c.k[page, off] = -127
    c.scales[0][page, :, off] = 1.0
    q = torch.ones((c.n, c.heads, 128), dtype=io, device="cuda")
    _, clean = run_attend(l2, c, io, q=q, window=window)
    c.scales[1][page, :, off] = value
    _, out = run_attend(l2, c, io, q=q, window=window)
    first = j - (200 - tokens)  # the position's own row
    assert clean.isfinite().all() and (not window or tokens - first <= window)  # (all rows from there on see it)
    assert torch.equal(out[:first], clean[:first]) and out[first:].isnan().all()


# a window that leaves nothing out, up to the largest number ("no limit"): the bits of no window, for rows of negative positions beside others too
@pytest.mark.parametrize("rows,kv,group", [([600, 1, 3], [5, 0, 0], 2), ([300, 70], [40, 69], 1), ([9, 1], [4, 2], 1), ([1, 1, 4], [300, 17, 90], 4), ([200, 140], [333, 140], 2)])
@pytest.mark.parametrize("cache,io", CACHES)
def test_windows_as_wide_as_the_table(l2, cache, io, rows, kv, group):
    c = Case(rows, kv, cache=cache, group=group, seed=12)
    room = c.table.shape[1] * c.page
    q, want = run_attend(l2, c, io)
    compare(l2, c, io, q=q)
    for window in (room, room + 1, 1 << 30, (1 << 31) - 1):
        for sinks in (0, 4, (1 << 31) - 1):
            assert torch.equal(run_attend(l2, c, io, q=q, window=window, sinks=sinks)[1], want), (window, sinks)
    for window, sinks in ((room - 1, 0), (max(kv), 3), (max(kv) - 1, (1 << 31) - 1)):
        compare(l2, c, io, q=q, window=window, sinks=sinks, what="window %d" % window)
    assert int(c.status) == 0


def test_launches_of_several_threads_are_counted(l2):
    """Threads with pages and streams of their own, side by side inside the library (a foreign call gives up the interpreter's lock)."""
    import threading
    calls, n_threads = 5000, 8
    own = []
    for i in range(n_threads):
        c = Case([1], [9], seed=i)
        pages, batch = c.handles(l2)
        rows = [torch.zeros((1, 2, 128), dtype=F16, device="cuda") for _ in "kv"]
        pages.read(batch, *rows)  # (fills the row records)
        own.append((pages, batch, rows, c, torch.cuda.Stream()))
    torch.cuda.synchronize()
    start, failed = threading.Barrier(n_threads), []

    def work(pages, batch, stream):
        start.wait()
        for _ in range(calls):
            if l2.lib.l2_kv_read(pages._ref, batch._ref, pages._at[0], pages._at[1], stream):
                failed.append(1)

    before = l2.lib.l2_launch_count()
    threads = [threading.Thread(target=work, args=(p, b, s.cuda_stream)) for p, b, _, _, s in own]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and l2.lib.l2_launch_count() - before == calls * n_threads


# a step said to have no rows that does bring some: left out and reported, as any that brings more than it says
@pytest.mark.parametrize("cache,io", CACHES)
def test_rows_of_a_step_that_says_it_has_none(l2, cache, io):
    from llama2_rs import paged
    c = Case([2, 1], [30, 40], cache=cache)
    pages, batch = c.handles(l2, max_rows=0)
    q = torch.ones((3, 2, 128), dtype=io, device="cuda")
    out = torch.full_like(q, 7.0)
    pages.attend(batch, q, out)
    assert (out == 7.0).all() and int(c.status) == paged.BAD_ROWS
    c = Case([0, 0], [30, 40], cache=cache, spare_rows=3)
    pages, batch = c.handles(l2)
    pages.attend(batch, q, out)
    assert (out == 7.0).all() and int(c.status) == 0

"""What the paged cache's entry points refuse before they look at a device (no GPU needed)."""
import ctypes as C

import pytest

A = 1 << 20  # an address on a 16-byte boundary that nothing reads: every call here is refused, or has no rows


def pages(l2, **kw):
    f = dict(k=A, v=A, k_scale=None, v_scale=None, page_stride=16 * 2 * 128, position_stride=2 * 128, head_stride=128, type=1, n_pages=4, page_size=16, n_kv_heads=2, head_size=128)
    f.update(kw)
    return l2._lib.KvPagesArgs(**f)


def batch(l2, **kw):
    f = dict(page_table=A, kv_len=A, row_start=A, status=None, n_seqs=2, table_width=3, n_rows=5, max_rows=4)
    f.update(kw)
    return l2._lib.KvBatchArgs(**f)


def rows(l2, **kw):
    f = dict(data=A, row_stride=256, head_stride=128, type=1, heads=2)
    f.update(kw)
    return l2._lib.KvRowsArgs(**f)


def ref(x):
    return C.byref(x) if x is not None else None


def append(l2, p, b, k, v, q=None, q_out=None, cos=None, sin=None, n=0):
    return l2.lib.l2_kv_append(ref(p), ref(b), ref(k), ref(v), ref(q), ref(q_out), cos, sin, n, None)


def attend(l2, p, b, q, out, scale=1.0, window=0, sinks=0, work=None, size=0):
    return l2.lib.l2_kv_attend(ref(p), ref(b), ref(q), ref(out), scale, window, sinks, work, size, None)


BAD_PAGES = [dict(type=0), dict(type=4), dict(head_size=96), dict(page_size=24), dict(page_size=4), dict(page_size=512), dict(n_pages=0), dict(n_kv_heads=0), dict(n_kv_heads=2000),
             dict(k=None), dict(v=A + 2), dict(page_stride=4), dict(position_stride=252), dict(head_stride=-128), dict(position_stride=64), dict(head_stride=64), dict(type=3),
             dict(type=3, k_scale=A, v_scale=A + 4), dict(page_stride=1 << 40)]
BAD_BATCH = [dict(n_seqs=-1), dict(n_rows=-1), dict(max_rows=-1), dict(table_width=-1), dict(n_seqs=70000), dict(kv_len=None), dict(row_start=None), dict(page_table=None)]
BAD_ROWS = [dict(type=3), dict(type=-1), dict(heads=3), dict(data=None), dict(data=A + 4), dict(row_stride=100), dict(head_stride=100), dict(row_stride=-256)]


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_pages(l2, bad):
    p, b, r = pages(l2, **bad), batch(l2), rows(l2)
    assert append(l2, p, b, r, r) == -1 and l2.lib.l2_kv_read(ref(p), ref(b), ref(r), ref(r), None) == -1 and attend(l2, p, b, r, r, work=A, size=1 << 30) == -1
    assert l2.lib.l2_kv_attend_workspace_bytes(ref(p), ref(b), 2) == 0 and l2.lib.l2_last_error()


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_batches(l2, bad):
    p, b, r = pages(l2), batch(l2, **bad), rows(l2)
    assert append(l2, p, b, r, r) == -1 and l2.lib.l2_kv_read(ref(p), ref(b), ref(r), ref(r), None) == -1 and attend(l2, p, b, r, r, work=A, size=1 << 30) == -1


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_rows(l2, bad):
    p, b, r, x = pages(l2), batch(l2), rows(l2), rows(l2, **bad)
    for k, v in ((x, r), (r, x)):
        assert append(l2, p, b, k, v) == -1 and l2.lib.l2_kv_read(ref(p), ref(b), ref(k), ref(v), None) == -1 and attend(l2, p, b, k, v, work=A, size=1 << 30) == -1


def test_what_does_not_go_together(l2):
    p, b, r = pages(l2), batch(l2), rows(l2)
    for missing in ((None, b, r, r), (p, None, r, r), (p, b, None, r), (p, b, r, None)):
        assert append(l2, *missing) == -1 and attend(l2, *missing, work=A, size=1 << 30) == -1 and l2.lib.l2_kv_read(*(ref(x) for x in missing), None) == -1
    assert append(l2, p, b, r, r, q=r) == -1                                    # q without q_out
    assert append(l2, p, b, r, r, q=rows(l2, heads=0), q_out=rows(l2, heads=0)) == -1
    assert append(l2, p, b, r, r, q=r, q_out=rows(l2, heads=4)) == -1
    assert append(l2, p, b, r, r, cos=A) == -1                                  # half a rope table
    assert append(l2, p, b, r, r, cos=A, sin=A, n=0) == -1
    assert append(l2, p, b, r, r, cos=A + 4, sin=A, n=9) == -1
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(sinks=-1)):
        assert attend(l2, p, b, r, r, work=A, size=1 << 30, **bad) == -1, bad
    assert attend(l2, p, b, rows(l2, type=2), rows(l2, type=2), work=A, size=1 << 30) == -1  # bf16 queries, f16 cache
    assert attend(l2, p, b, rows(l2, type=0), r, work=A, size=1 << 30) == -1                 # f32 queries
    assert attend(l2, p, b, r, rows(l2, type=2), work=A, size=1 << 30) == -1                 # an output of another type
    assert attend(l2, p, b, rows(l2, heads=3), rows(l2, heads=3), work=A, size=1 << 30) == -1
    assert attend(l2, p, b, rows(l2, heads=2 * 65), rows(l2, heads=2 * 65), work=A, size=1 << 30) == -1


def test_sizes_out_of_range(l2):
    r = rows(l2)
    assert append(l2, pages(l2), batch(l2, table_width=1 << 27), r, r) == -5
    assert attend(l2, pages(l2), batch(l2, table_width=1 << 26, max_rows=1 << 29), r, r, work=A, size=1 << 30) == -5


def test_no_device(l2):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    p, b, r = pages(l2), batch(l2, n_rows=0), rows(l2)
    assert append(l2, p, b, r, r) == -3 and l2.lib.l2_kv_read(ref(p), ref(b), ref(r), ref(r), None) == -3 and attend(l2, p, b, r, r) == -3
    assert l2.lib.l2_kv_attend_workspace_bytes(ref(p), ref(b), 2) == 0 and b"no CPU fallback" in l2.lib.l2_last_error()

"""What l2_kv_plan, l2_kv_release and l2_block_norm refuse before they look at a device (no GPU needed)."""
import ctypes as C

import pytest

A = 1 << 20  # an address that nothing reads: every call here is refused, or has no device


def tables(l2, **kw):
    f = dict(page_table=A, kv_len=A, free_pages=A, free_count=A, status=None, n_seqs=3, table_width=8, n_pages=20, page_size=16)
    f.update(kw)
    return l2._lib.KvTablesArgs(**f)


def plan(l2, t, new=A, start=A, slots=A, positions=A, n_rows=10, max_rows=4):
    return l2.lib.l2_kv_plan(C.byref(t) if t is not None else None, new, start, slots, positions, n_rows, max_rows, None)


def release(l2, t, keep=A, window=0, sinks=0):
    return l2.lib.l2_kv_release(C.byref(t) if t is not None else None, keep, window, sinks, None)


BAD_TABLES = [dict(page_size=0), dict(page_size=24), dict(page_size=4), dict(page_size=512), dict(n_seqs=-1), dict(n_seqs=16385), dict(table_width=-1), dict(n_pages=0), dict(free_pages=None),
              dict(free_count=None), dict(kv_len=None), dict(page_table=None), dict(kv_len=A + 2), dict(status=A + 1), dict(free_pages=A + 3)]


@pytest.mark.parametrize("bad", BAD_TABLES)
def test_tables(l2, bad):
    assert plan(l2, tables(l2, **bad)) == -1 and release(l2, tables(l2, **bad)) == -1 and l2.lib.l2_last_error()


def test_arguments(l2):
    t = tables(l2)
    for bad in (dict(new=None), dict(start=None), dict(n_rows=-1), dict(max_rows=-1), dict(n_rows=(1 << 30) + 1), dict(slots=A + 4), dict(positions=A + 2), dict(new=A + 1), dict(start=A + 2)):
        assert plan(l2, t, **bad) == -1, bad
    for bad in (dict(window=-1), dict(sinks=-1), dict(keep=A + 2)):
        assert release(l2, t, **bad) == -1, bad
    assert plan(l2, None) == -1 and release(l2, None) == -1
    assert plan(l2, tables(l2, table_width=1 << 20, n_seqs=1 << 11)) == -5
    assert plan(l2, tables(l2, table_width=1 << 27)) == -5 and release(l2, tables(l2, table_width=1 << 27)) == -5


def norm(l2, **kw):
    rows = lambda data=A, stride=64, type=0: l2._lib.RowsArgs(data, stride, type)  # noqa: E731
    f = dict(block=rows(), residual=rows(A + (1 << 16)), gate=rows(None), residual_out=rows(A + (2 << 16)), out=rows(A + (3 << 16)), post_weight=None, pre_weight=None, scale=1.0, eps=1e-5, rows=3, dim=64)
    for name, value in kw.items():
        f[name] = rows(*value) if isinstance(value, tuple) else value
    return l2.lib.l2_block_norm(C.byref(l2._lib.BlockNormArgs(**f)), None)


BAD_NORMS = [dict(rows=-1), dict(dim=0), dict(dim=32769), dict(dim=-4), dict(block=(A, 64, 3)), dict(residual=(A, 64, 4)), dict(gate=(A, 64, -1)), dict(out=(A + (3 << 16), 64, 9)), dict(block=(A + 2, 64, 0)),
             dict(block=(A + 1, 64, 1)), dict(block=(A, -64, 0)), dict(residual=(A, 1 << 41, 0)), dict(out=(A + (3 << 16), 63, 0)), dict(residual_out=(A + (2 << 16), 0, 0)),
             dict(block=(None, 0, 0), residual=(None, 0, 0)), dict(out=(None, 0, 0), residual_out=(None, 0, 0)), dict(block=(None, 0, 0), gate=(A, 0, 1)), dict(block=(None, 0, 0), post_weight=A),
             dict(eps=-1e-9), dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("nan")), dict(scale=float("-inf")), dict(post_weight=A + 2), dict(pre_weight=A + 1),
             # results on one another, or on what is read in another order
             dict(residual_out=(A + (3 << 16) + 4 * 190, 64, 0)), dict(out=(A + (1 << 16), 64, 0)), dict(residual_out=(A, 64, 0)), dict(out=(A, 64, 1)), dict(out=(A + 4, 64, 0)), dict(out=(A, 65, 0)),
             dict(residual_out=(A + (1 << 16), 64, 2)), dict(gate=(A + (3 << 16), 0, 0)), dict(pre_weight=A + (3 << 16) + 4 * 100), dict(post_weight=A + (2 << 16) - 4 * 63)]


@pytest.mark.parametrize("bad", BAD_NORMS)
def test_norms(l2, bad):
    assert norm(l2, **bad) == -1 and l2.lib.l2_last_error()


def test_what_is_right_reaches_the_device(l2):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    assert plan(l2, tables(l2)) == -3 and release(l2, tables(l2)) == -3 and release(l2, tables(l2), keep=None) == -3 and plan(l2, tables(l2), slots=None, positions=None) == -3
    for fine in (dict(), dict(out=(A, 64, 0)), dict(residual_out=(A + (1 << 16), 64, 0)), dict(gate=(A + (5 << 16), 0, 2)), dict(block=(A, 0, 0)), dict(rows=0), dict(out=(None, 0, 0)),
                 dict(residual_out=(None, 0, 0)), dict(block=(None, 0, 0)), dict(residual=(None, 0, 0)), dict(block=(A + 4, 67, 0))):
        assert norm(l2, **fine) == -3, fine
    assert b"no CPU fallback" in l2.lib.l2_last_error()

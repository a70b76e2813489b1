"""What the paged cache's entry points refuse of a cache in 4 bits before they look at a device (no GPU needed)."""
import ctypes as C

import pytest

from test_paged_arguments import A, append, attend, batch, ref, rows
from test_paged_arguments import pages as pages_of


def pages(l2, **kw):
    return pages_of(l2, **{**dict(type=4, k_scale=A, v_scale=A), **kw})


BAD_PAGES = [dict(k_scale=None), dict(v_scale=None), dict(k_scale=A + 4), dict(v_scale=A + 8), dict(type=5), dict(type=-1), dict(head_size=96), dict(head_size=256), dict(page_size=12),
             dict(page_stride=16 * 2 * 128 + 16), dict(position_stride=2 * 128 + 8), dict(head_stride=144), dict(head_stride=64), dict(position_stride=128), dict(k=A + 8), dict(head_stride=0)]


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_pages(l2, bad):
    p, b, r = pages(l2, **bad), batch(l2), rows(l2)
    assert append(l2, p, b, r, r) == -1 and l2.lib.l2_kv_read(ref(p), ref(b), ref(r), ref(r), None) == -1 and attend(l2, p, b, r, r, work=A, size=1 << 30) == -1
    assert l2.lib.l2_kv_attend_workspace_bytes(ref(p), ref(b), 2) == 0 and l2.lib.l2_last_error()


def test_queries(l2):
    p, b = pages(l2), batch(l2)
    assert attend(l2, p, b, rows(l2, type=0), rows(l2), work=A, size=1 << 30) == -1           # f32 queries
    assert attend(l2, p, b, rows(l2, type=2), rows(l2, type=1), work=A, size=1 << 30) == -1   # an output of another type
    assert attend(l2, p, b, rows(l2, type=4), rows(l2, type=4), work=A, size=1 << 30) == -1   # rows of 4 bits
    assert append(l2, p, b, rows(l2, type=4), rows(l2)) == -1


def test_what_is_right_reaches_the_device(l2):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    p, b, r = pages(l2, head_stride=160, position_stride=2 * 160, page_stride=16 * 2 * 160), batch(l2, n_rows=0), rows(l2)
    for q in (r, rows(l2, type=2)):
        assert attend(l2, p, b, q, q, work=A, size=1 << 30) == -3
    assert append(l2, p, b, r, r) == -3 and l2.lib.l2_kv_read(ref(p), ref(b), ref(r), ref(r), None) == -3
    assert C.sizeof(type(p)) == 80

"""Attention over a cache in 4 bits may read its queries again behind its first results: an output on them is refused (no GPU needed)."""
import pytest

from test_paged4_arguments import pages
from test_paged_arguments import A, attend, batch, rows
from test_paged_arguments import pages as pages_of


def call(l2, q, out, p=None, **kw):
    return attend(l2, p or pages(l2), batch(l2, **kw), rows(l2, **{"data": A + (1 << 16), **q}), rows(l2, **{"data": A + (1 << 16), **out}), work=A, size=1 << 30)


# five rows of two heads of 128 in 16 bits: 256 elements a row, 2560 bytes in all
@pytest.mark.parametrize("q,out", [(dict(), dict()), (dict(), dict(type=0)), (dict(), dict(data=A + (1 << 16) + 2544)), (dict(data=A + (1 << 16) + 16), dict()),
                                   (dict(row_stride=512), dict(row_stride=512, data=A + (1 << 16) + 256)), (dict(row_stride=512), dict(data=A + (1 << 16) + 512)),
                                   (dict(row_stride=128, head_stride=640), dict(row_stride=128, head_stride=640)), (dict(row_stride=0, data=A + (1 << 16) + 1024), dict())])
def test_refused(l2, q, out):
    assert call(l2, q, out) == -1 and b"out" in l2.lib.l2_last_error()


@pytest.mark.parametrize("q,out", [(dict(), dict(data=A + (1 << 16) + 2560)), (dict(data=A + (1 << 16) + 2560), dict()),
                                   (dict(row_stride=512), dict(row_stride=512, data=A + (1 << 16) + 512)),     # halves of one array's rows
                                   (dict(row_stride=512, data=A + (1 << 16) + 512), dict(row_stride=512)),
                                   (dict(row_stride=128, head_stride=1280), dict(row_stride=128, head_stride=1280, data=A + (1 << 16) + 1280)),  # head by head, in turn
                                   (dict(row_stride=0, data=A + (1 << 16) + 512), dict(row_stride=768))])      # one row of queries in the gaps
def test_apart(l2, q, out):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    assert call(l2, q, out) == -3


def test_other_caches_and_calls_without_rows(l2):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    assert call(l2, {}, {}, p=pages_of(l2)) == -3 and call(l2, {}, {}, n_rows=0) == -3

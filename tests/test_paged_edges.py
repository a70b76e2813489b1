"""What the paged cache's entry points and objects refuse at the edges of their ranges (no GPU needed)."""
import pytest

from test_paged_arguments import A, append, attend, batch, pages, ref, rows


# the size of a workspace is asked for before attention itself checks anything: heads that no kernel takes must not reach its divisions
@pytest.mark.parametrize("heads,kv_heads", [(65, 1), (130, 2), (256, 1), (257, 1), (1 << 20, 1), (3, 2), (0, 1), (-2, 2)])
def test_workspace_of_heads_out_of_range(l2, heads, kv_heads):
    p, b = pages(l2, n_kv_heads=kv_heads), batch(l2)
    assert l2.lib.l2_kv_attend_workspace_bytes(ref(p), ref(b), heads) == 0
    assert b"query heads" in l2.lib.l2_last_error()
    r = rows(l2, heads=heads)
    assert attend(l2, p, b, r, r, work=A, size=1 << 30) == -1 and b"query heads" in l2.lib.l2_last_error()


def test_workspace_of_too_many_tiles(l2):
    p, b = pages(l2), batch(l2, table_width=1 << 26, max_rows=1 << 29)
    assert l2.lib.l2_kv_attend_workspace_bytes(ref(p), ref(b), 2) == 0 and b"2^31 tiles" in l2.lib.l2_last_error()


def test_workspace_in_python(l2):
    stand_in = pytest.importorskip("stand_in")
    for heads in (3, 130, 514):
        with pytest.raises(l2.L2Error, match="query heads"):
            stand_in.pages(l2).workspace_bytes(stand_in.batch(l2), heads)


# ctypes cuts numbers to 32 bits: a window of 2^32 + 5 would be a window of 5
@pytest.mark.parametrize("wide", [1 << 31, (1 << 32) + 5, -(1 << 31) - 1, 1 << 70])
def test_numbers_beyond_32_bits(l2, wide):
    stand_in = pytest.importorskip("stand_in")
    torch = stand_in.torch
    pages, batch = stand_in.pages(l2), stand_in.batch(l2)
    q = stand_in.tensor((5, 2, 128), torch.float16)
    work = stand_in.tensor((1 << 20,), torch.uint8)
    for bad in (lambda: pages.attend(batch, q, q, window=wide, workspace=work, stream=0), lambda: pages.attend(batch, q, q, window=9, sinks=wide, workspace=work, stream=0),
                lambda: stand_in.batch(l2, rows=wide), lambda: stand_in.batch(l2, most=wide), lambda: pages.workspace_bytes(batch, wide)):
        with pytest.raises(ValueError, match="beyond 32 bits"):
            bad()


def test_sizes_beyond_32_bits(l2):
    stand_in = pytest.importorskip("stand_in")
    for bad in (lambda: stand_in.pages(l2, n_pages=1 << 32), lambda: stand_in.pages(l2, heads=(1 << 32) + 2), lambda: stand_in.batch(l2, width=(1 << 32) + 3)):
        with pytest.raises(ValueError, match="beyond 32 bits"):
            bad()


# pages, batch and launch belong to one device: the table and lengths of another would be read (and its status word written) there
@pytest.mark.parametrize("pages_on,batch_on,current", [(0, 1, 0), (1, 0, 1), (1, 1, 0), (0, 0, 1)])
@pytest.mark.parametrize("stream", [None, 1234])
def test_one_device(l2, monkeypatch, stream, pages_on, batch_on, current):
    stand_in = pytest.importorskip("stand_in")
    torch = stand_in.torch
    from llama2_rs import paged

    def launched(*args):
        raise AssertionError("a launch")

    monkeypatch.setattr(paged, "_cuda", (lambda: current, lambda device: 0))
    for call in ("_append", "_read", "_attend"):
        monkeypatch.setattr(paged, call, launched)
    pages, batch = stand_in.pages(l2, pages_on), stand_in.batch(l2, batch_on)
    x, work = stand_in.tensor((5, 2, 128), torch.float16, pages_on), stand_in.tensor((1 << 20,), torch.uint8, pages_on)
    for bad in (lambda: pages.append(batch, x, x, stream=stream), lambda: pages.read(batch, x, x, stream=stream),
                lambda: pages.attend(batch, x, x, workspace=work, stream=stream)):
        with pytest.raises(ValueError, match="device"):
            bad()
    monkeypatch.setattr(paged, "_cuda", (lambda: pages_on, lambda device: 0))
    with pytest.raises(AssertionError, match="a launch"):  # (all on one device)
        pages.append(stand_in.batch(l2, pages_on), x, x, stream=stream)


def test_rotation_out_of_range(l2):
    p, b, r = pages(l2), batch(l2), rows(l2)
    for rotation in (-1, 2):
        assert l2.lib.l2_kv_append_rope(ref(p), ref(b), ref(r), ref(r), None, None, A, A, 9, rotation, None) == -1 and b"rotation" in l2.lib.l2_last_error()


# a pool of 4 pages of 16 positions and 2 heads of 128: what would lie on one another is refused, whatever dimension it is
@pytest.mark.parametrize("strides", [(4096, 128, 128), (4096, 256, 144), (4000, 256, 128), (128, 1024, 256), (256, 256, 128), (4096, 256, 256), (128, 2048, 128), (2048, 128, 2048)])
def test_pools_that_overlap(l2, strides):
    p, b, r = pages(l2, **dict(zip(("page_stride", "position_stride", "head_stride"), strides))), batch(l2), rows(l2)
    assert append(l2, p, b, r, r) == -1 and b"overlap" in l2.lib.l2_last_error()


# page by page, head by head, position by position, with gaps: all of these are pools
@pytest.mark.parametrize("strides", [(4096, 256, 128), (4096, 128, 2048), (128, 512, 8192), (128, 1024, 512), (4160, 256, 128), (4352, 272, 136), (256, 1024, 128)])
def test_pools_that_do_not(l2, strides):
    p, b = pages(l2, **dict(zip(("page_stride", "position_stride", "head_stride"), strides))), batch(l2)
    r = rows(l2, heads=3)  # (refused for its heads, after the pool has been looked at)
    assert append(l2, p, b, r, r) == -1 and b"3 heads" in l2.lib.l2_last_error()


# several rows written to one place: refused; read from one place: not
@pytest.mark.parametrize("bad", [dict(row_stride=0), dict(row_stride=128), dict(head_stride=64), dict(head_stride=0), dict(row_stride=64, head_stride=320), dict(row_stride=128, head_stride=512)])
def test_written_rows_that_overlap(l2, bad):
    p, b, r, x = pages(l2), batch(l2), rows(l2), rows(l2, **bad)
    for call in (lambda: l2.lib.l2_kv_read(ref(p), ref(b), ref(x), ref(r), None), lambda: l2.lib.l2_kv_read(ref(p), ref(b), ref(r), ref(x), None),
                 lambda: append(l2, p, b, r, r, q=r, q_out=x), lambda: attend(l2, p, b, r, x, work=A, size=1 << 30)):
        assert call() == -1 and b"overlap" in l2.lib.l2_last_error()
    assert append(l2, p, b, x, x, q=x, q_out=rows(l2, row_stride=100)) == -1 and b"q_out has strides" in l2.lib.l2_last_error()  # (k, v and q went through)

"""Arrays of l2_block_norm that lie between one another's rows (no GPU needed)."""
import pytest

from test_tables_norm_arguments import A, norm

B, C = A + (2 << 16), A + (1 << 16)  # where results begin; the residual

# three rows of 64 elements of f32: 256 bytes
FINE = [dict(residual_out=(B, 128, 0), out=(B + 256, 128, 0)), dict(residual_out=(B + 256, 128, 0), out=(B, 128, 0)), dict(residual_out=(B, 100, 0), out=(B + 272, 200, 1)) | dict(rows=1),
        dict(block=(B, 128, 0), out=(B + 256, 128, 0), residual_out=(None, 0, 0)), dict(residual=(B + 256, 192, 0), residual_out=(B, 192, 0), gate=(B + 512, 192, 0)),
        dict(residual_out=(B, 128, 0), gate=(B + 256, 0, 0)), dict(residual_out=(B, 128, 0), pre_weight=B + 768), dict(residual_out=(B, 128, 0), out=(B + 256, 256, 2)),
        dict(residual_out=(B, 96, 0), out=(B + 256, 192, 1))]
BAD = [dict(residual_out=(B, 128, 0), out=(B + 252, 128, 0)), dict(residual_out=(B, 128, 0), out=(B + 260, 128, 0)), dict(residual_out=(B, 128, 0), out=(B + 256, 129, 0)),
       dict(residual_out=(B, 127, 0), out=(B + 256, 127, 0)), dict(residual_out=(B, 128, 0), gate=(B + 260, 0, 0)), dict(residual_out=(B, 128, 0), pre_weight=B + 764),
       dict(residual_out=(B, 128, 0), out=(B + 256, 128, 1)), dict(block=(B + 128, 128, 0), out=(B, 128, 0)), dict(residual_out=(B, 1 << 40, 0), out=(B + 256, (1 << 40) - 4, 0), rows=1 << 30)]


@pytest.mark.parametrize("bad", BAD)
def test_refused(l2, bad):
    assert norm(l2, **bad) == -1 and b"overlap" in l2.lib.l2_last_error()


@pytest.mark.parametrize("fine", FINE)
def test_apart(l2, fine):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    assert norm(l2, **fine) == -3, l2.lib.l2_last_error()

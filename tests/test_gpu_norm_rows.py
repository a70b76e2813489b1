"""Norms: rows as many as 31 bits count."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_block_norm import BF16, F16  # noqa: E402


def test_as_many_rows_as_there_can_be(l2):
    rows = (1 << 31) - 1
    block = torch.tensor([[3.0]], dtype=BF16, device="cuda").expand(rows, 1)
    out = torch.zeros((rows, 1), dtype=F16, device="cuda")
    l2.block_norm(block, None, out, eps=7.0)
    exact = 0.75  # 3 / sqrt(9 + 7)
    for i in range(0, rows, 1 << 28):
        assert bool((out[i:i + (1 << 28)] == exact).all())

"""Norms: rows as many as 31 bits count, and results between one another's rows."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_block_norm import BF16, F16, F32, check, make, run, want  # noqa: E402


def test_as_many_rows_as_there_can_be(l2):
    rows = (1 << 31) - 1
    block = torch.tensor([[3.0]], dtype=BF16, device="cuda").expand(rows, 1)
    out = torch.zeros((rows, 1), dtype=F16, device="cuda")
    l2.block_norm(block, None, out, eps=7.0)
    exact = 0.75  # 3 / sqrt(9 + 7)
    for i in range(0, rows, 1 << 28):
        assert bool((out[i:i + (1 << 28)] == exact).all())


@pytest.mark.parametrize("rows,dim", [(1, 640), (37, 640), (900, 130), (700, 515)])
def test_results_side_by_side(l2, rows, dim):
    """Both results, and what is read, as parts of one array's rows."""
    a = make(rows, dim, F32, F32, gate=("channel", F32))
    plain = run(l2, a, out=F32, residual_out=F32)
    room = torch.full((rows, 4, dim), 9.0, device="cuda")
    room[:, 1], room[:, 3] = a["block"], a["residual"]
    l2.block_norm(room[:, 1], room[:, 3], room[:, 2], residual_out=room[:, 0], post_weight=a["post_weight"], pre_weight=a["pre_weight"], gate=a["gate"])
    er, sr, eo, so = want(a, 1.0, 1e-5)
    check(room[:, 0], er, sr), check(room[:, 2], eo, so)
    assert torch.equal(room[:, 1], a["block"]) and torch.equal(room[:, 3], a["residual"])
    if dim % 4 == 0:
        assert torch.equal(room[:, 0], plain[0]) and torch.equal(room[:, 2], plain[1])

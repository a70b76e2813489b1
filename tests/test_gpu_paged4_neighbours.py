"""Attention over a cache in 4 bits for few rows: a row's result goes by what the row sees, whatever the rows beside it bring and the rest of a page holds."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged4_reference import Case4, attend4  # noqa: E402
from paged_reference import check  # noqa: E402
from test_gpu_paged4 import BF16, F16, F32, run_attend  # noqa: E402
from test_gpu_paged4_rows import only  # noqa: E402


def stairs(tokens, group, kv_heads, value=None):
    """Sequences enough that a CTA takes them whole, in several steps.  K equal in all elements of a position: 0, and 10 at the last five, where V is small; `value` for the scales behind."""
    n = 320
    kv = torch.randint(990, 1006, (n,), generator=torch.Generator().manual_seed(1)).tolist()
    c = Case4([tokens] * n, kv, group=group, kv_heads=kv_heads, seed=5)
    c.scales[0].zero_()
    for b in range(n):
        for j in range(kv[b] - 5, -(-kv[b] // 16) * 16):
            page, off = c.slot(b, j)
            if j < kv[b]:
                c.scales[0][page, :, off, 1] = 10.1
                c.scales[1][page, :, off] = (c.scales[1][page, :, off].float() * 2.0**-10).to(BF16)
            elif value is not None:
                c.scales[0][page, :, off, 0] = c.scales[1][page, :, off, 0] = value
    return c


@pytest.mark.parametrize("value", [float("inf"), float("nan"), 3.0e38])
@pytest.mark.parametrize("tokens,group,kv_heads", [(1, 1, 4), (1, 5, 2), (2, 3, 1), (3, 4, 4)])
def test_the_rest_of_the_last_page_does_not_matter(l2, tokens, group, kv_heads, value):
    """Few rows: positions behind the last may have any scale, also where the scores of the last positions rise."""
    c = stairs(tokens, group, kv_heads)
    q = torch.zeros((c.n, c.heads, 128), dtype=BF16, device="cuda")
    q[:, :, 0] = 1
    _, clean = run_attend(l2, c, BF16, scale=1.0, q=q, out_type=F32)
    _, out = run_attend(l2, stairs(tokens, group, kv_heads, value), BF16, scale=1.0, q=q, out_type=F32)
    assert torch.equal(out, clean) and out.isfinite().all()


# kv heads: four warps to a head, two, and one
@pytest.mark.parametrize("kv_heads", [1, 2, 4])
@pytest.mark.parametrize("group", [2, 7, 12])
@pytest.mark.parametrize("io", [F16, BF16])
def test_a_row_does_not_follow_its_neighbours_scores(l2, io, group, kv_heads):
    """Few rows: one row's scores rise so far that what it has summed is scaled; the rows beside it rise less, and keep their bits whether it does or not."""
    c = stairs(1, group, kv_heads)
    q = torch.zeros((c.n, c.heads, 128), dtype=io, device="cuda")
    q[:, :, 0] = 1
    rising = q.clone()
    rising[:, ::group, 0] = 16
    outs = [run_attend(l2, c, io, scale=1.0, q=x, out_type=F32)[1] for x in (q, rising)]
    keep = torch.arange(c.heads) % group != 0
    assert torch.equal(outs[0][:, keep], outs[1][:, keep])
    part = only(c, range(7))
    for x, out in zip((q, rising), outs):
        want, bound = attend4(part, x, 1.0)
        check(out[:7], want[:7], bound[:7])

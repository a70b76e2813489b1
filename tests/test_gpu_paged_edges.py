"""The paged cache and its attention at the edges of what they are given."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged_reference import Case  # noqa: E402
from test_gpu_paged import BF16, F16, I8, compare  # noqa: E402


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

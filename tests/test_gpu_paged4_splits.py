"""Attention over a cache in 4 bits for few rows, with kv heads that CTAs share in every way: four, two or one a CTA, one to three of these a sequence."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged4_reference import Case4, attend4  # noqa: E402
from paged_reference import check  # noqa: E402
from test_gpu_paged4 import BF16, F16, F32, compare, run_attend  # noqa: E402

HEADS = [4, 8, 12, 6, 3]


@pytest.mark.parametrize("kv_heads", HEADS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("io", [F16, BF16])
def test_single_tokens_and_drafts(l2, io, hd, kv_heads):
    kv = [1, 2, 16, 17, 63, 64, 65, 0, 128, 129, 256, 300, 555, 31]
    rows = [1] * len(kv)
    rows[-1] = 0
    for group in (1, 8, 16):
        compare(l2, Case4(rows, kv, hd=hd, group=group, kv_heads=kv_heads, seed=group), io, what="tokens %d" % group)
    for group in (1, 3, 5):
        compare(l2, Case4([2, 0, 1, 3], [260, 5, 700, 129], hd=hd, group=group, kv_heads=kv_heads, seed=group, layout="HND", page=32, spare_rows=2), io, what="drafts %d" % group)


@pytest.mark.parametrize("kv_heads", HEADS)
@pytest.mark.parametrize("window,sinks", [(5, 3), (100, 64), (300, 4), (40, 1000)])
def test_window_and_sinks(l2, window, sinks, kv_heads):
    for group in (2, 4):
        compare(l2, Case4([1, 1, 1, 4, 1], [1, 64, 900, 300, 2500], group=group, kv_heads=kv_heads, seed=window), BF16, window=window, sinks=sinks)


# one sequence in many pieces, alone and among short ones
@pytest.mark.parametrize("kv_heads", HEADS)
@pytest.mark.parametrize("hd,tokens,group", [(128, 1, 1), (64, 1, 8), (128, 2, 8), (64, 3, 3)])
def test_pieces(l2, hd, tokens, group, kv_heads):
    compare(l2, Case4([tokens], [9001], hd=hd, group=group, kv_heads=kv_heads, page=64), BF16, what="alone")
    compare(l2, Case4([1, 1, tokens, 1, 0, 1], [30, 1, 7007, 200, 9, 64], hd=hd, group=group, kv_heads=kv_heads, page=8), BF16, what="among others")


@pytest.mark.parametrize("kv_heads", HEADS)
def test_many_sequences(l2, kv_heads):
    g = torch.Generator().manual_seed(kv_heads)
    kv = torch.randint(0, 150, (260,), generator=g).tolist()
    compare(l2, Case4([int(x % 7 != 3) for x in kv], kv, group=4, hd=64, kv_heads=kv_heads), BF16)


# Rows of Q reach the products as f16, times a power of two that brings the largest element to 2^15 or more: elements of even index as they are, of odd index as a
# sixteenth.  Half of f16's smallest step, 2^-25, is then 2^-40 of the row's largest element for the one, 2^-36 for the other.
@pytest.mark.parametrize("kv_heads", [1, 2, 4])
@pytest.mark.parametrize("io", [F16, BF16])
def test_queries_of_tiny_elements_beside_a_huge_one(l2, io, kv_heads):
    c = Case4([1, 1], [3, 17], kv_heads=kv_heads, group=3, seed=2)
    c.k[..., 0] &= 0xf0           # nothing comes of the huge element (of index 0) ...
    c.scales[0][..., 0], c.scales[0][..., 1] = 1.0, 0.0
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.zeros((2, c.heads, 128), device="cuda")
    q[..., 1::2] = torch.rand((2, c.heads, 64), generator=g, device="cuda").sub_(0.5).mul_(2.0**-11)  # ... and all of it of the odd ones
    q[..., 0] = 2.0**15
    q = q.to(io)
    scale = 2.0**7
    _, out = run_attend(l2, c, io, scale=scale, q=q, out_type=F32)
    want, bound = attend4(c, q, scale)
    # a score is off by the rounding of 64 odd elements times u, and two scores move a probability by e to twice that, less one
    off = scale * 64 * 15 * 2.0**15 * 2.0**-36
    for b in range(2):
        u, s, z = c.numbers(1, b)
        sizes = (z.abs() + s.abs() * u).repeat_interleave(c.group, 1)
        k = c.cached(0, b).repeat_interleave(c.group, 1)
        w = torch.softmax(torch.einsum("hd,jhd->hj", q[b].double(), k) * scale, -1)
        bound[b] += math.expm1(2 * off) * torch.einsum("hj,jhd->hd", w, sizes)
    check(out, want, bound)

"""Attention over a cache in 4 bits: a row's result goes by what the row sees, whatever the others bring and see."""
import copy

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged4_reference import Case4, attend4  # noqa: E402
from paged_reference import check  # noqa: E402
from test_gpu_paged4 import BF16, F16, F32, run_attend  # noqa: E402

# pairs (scale, zero) that f16 does not hold: values beyond 65504, steps below 2^-16, a head of one small number
NOT_HELD = [(6000.0, 5.0), (0.25, 3.0e5), (2.0**-20, 2.0**-21), (0.0, 2.0**-20)]


def only(c, chosen):
    """The case with the rows of some of its sequences, for the 64-bit result of these alone."""
    x = copy.copy(c)
    x.rows = [n if b in chosen else 0 for b, n in enumerate(c.rows)]
    return x


def seen_from(c, b, j, window, sinks):
    """Of sequence b's rows, which see position j."""
    p = torch.arange(c.rows[b]) + c.kv[b] - c.rows[b]
    seen = p >= j
    return seen & ((p - j < window) | (j < sinks)) if window else seen


def mixed(c, q, scale, window, sinks):
    """(result, bound) where some of what a row sees goes through the products in bf16 and the rest in f16: an error is the one's or the other's."""
    want, wide = attend4(c, q, scale, window, sinks, many=True, wide=True)
    return want, wide + attend4(c, q, scale, window, sinks, many=True, wide=False)[1]


@pytest.mark.parametrize("pair", NOT_HELD)
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("io", [F16, BF16])
def test_values_that_f16_does_not_hold_and_rows_that_do_not_see_them(l2, io, which, pair):
    """One pair of one sequence: rows in front of it, behind its window, and of the other sequences keep their bits."""
    for rows, kv, hd, window, sinks, out_type, layout in (([200, 150, 3], [333, 150, 90], 128, 0, 0, None, "NHD"), ([200, 40], [333, 700], 64, 60, 4, F32, "HND"),
                                                          ([300, 129], [300, 400], 128, 100, 0, F32, "HND"), ([40, 300], [5000, 300], 128, 0, 0, None, "NHD")):
        c = Case4(rows, kv, group=2, hd=hd, seed=4, layout=layout)
        q, clean = run_attend(l2, c, io, window=window, sinks=sinks, out_type=out_type)
        for j in (kv[0] - rows[0] // 2, max(0, kv[0] - rows[0] - 20)):  # in the chunk, in front of it
            page, off = c.slot(0, j)
            before = c.scales[which][page, 1, off].clone()
            c.scales[which][page, 1, off] = torch.tensor(pair).to(BF16)  # (of one kv head)
            _, out = run_attend(l2, c, io, window=window, sinks=sinks, out_type=out_type, q=q)
            seen = torch.zeros(c.n, dtype=torch.bool)
            seen[:rows[0]] = seen_from(c, 0, j, window, sinks)
            assert seen.any() and int(c.status) == 0
            assert torch.equal(out[:, :2], clean[:, :2]), "the other kv head"
            assert torch.equal(out[~seen], clean[~seen]), (rows, j)
            if which == 1 or max(abs(x) for x in pair) < 1:  # (scores of 10^5 are no test of anything)
                part = only(c, [0])
                want, bound = mixed(part, q, hd**-0.5, window, sinks)
                check(out[seen], want[seen], bound[seen], str(j))
            else:
                assert out.isfinite().all()
            c.scales[which][page, 1, off] = before


def test_values_that_f16_does_not_hold_in_many_short_pieces(l2):
    """A few sequences of thousands, of which a CTA has more than it has bits for."""
    n = 6000
    c = Case4([9] * n, [int(x) for x in np.random.default_rng(1).integers(9, 14, n)], kv_heads=1, group=2, hd=64, page=8, seed=7)
    q, clean = run_attend(l2, c, BF16)
    chosen = [0, 1, 17, 35, 36, 40, 77, 2000, 2039, 3333, 4001, 5998, 5999]
    for i, b in enumerate(chosen):
        page, off = c.slot(b, c.kv[b] - 1 - i % 5)
        c.scales[i % 2][page, :, off] = torch.tensor((2.0**-20, 2.0**-21)).to(BF16)
    _, out = run_attend(l2, c, BF16, q=q)
    seen = torch.zeros(c.n, dtype=torch.bool)
    for i, b in enumerate(chosen):
        start = int(c.row_start[b])
        seen[start:start + 9] = seen_from(c, b, c.kv[b] - 1 - i % 5, 0, 0)
    assert torch.equal(out[~seen], clean[~seen])
    want, bound = mixed(only(c, chosen), q, 64**-0.5, 0, 0)
    check(out[seen], want[seen], bound[seen])


def test_values_that_f16_does_not_hold_beside_a_nan(l2):
    """Both in one sequence: rows that see the NaN are NaN, the others as if it were not there."""
    for which in (0, 1):
        c = Case4([200, 60], [333, 100], group=2, seed=4)
        page, off = c.slot(0, 200)
        c.scales[which][page, :, off] = torch.tensor((2.0**-20, 2.0**-21)).to(BF16)
        q, clean = run_attend(l2, c, BF16)
        page, off = c.slot(0, 250)
        c.scales[1][page, :, off, 0] = float("nan")
        _, out = run_attend(l2, c, BF16, q=q)
        seen = torch.zeros(c.n, dtype=torch.bool)
        seen[:200] = seen_from(c, 0, 250, 0, 0)
        assert out[seen].isnan().all() and torch.equal(out[~seen], clean[~seen])


def test_values_that_f16_does_not_hold_in_a_graph(l2):
    """Captured with values that f16 holds, replayed with others, and with the first again."""
    c = Case4([100, 60], [333, 100], group=2, seed=4)
    q = torch.randn((c.n, c.heads, 128), device="cuda").to(F16)
    out = torch.zeros_like(q)
    pages, batch = c.handles(l2)
    work = torch.empty(pages.workspace_bytes(batch, c.heads), dtype=torch.uint8, device="cuda")
    pages.attend(batch, q, out, workspace=work)
    torch.cuda.synchronize()
    clean = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.attend(batch, q, out, workspace=work)
    page, off = c.slot(0, 200)
    keep = c.scales[1][page, :, off].clone()
    for pair in ((2.0**-20, 2.0**-21), None, (0.0, 2.0**-20)):
        c.scales[1][page, :, off] = keep if pair is None else torch.tensor(pair, device="cuda").to(BF16)
        graph.replay()
        want, bound = mixed(only(c, [0]), q, 128**-0.5, 0, 0)
        check(out[:100], want[:100], bound[:100])
        assert torch.equal(out[100:], clean[100:]) and (pair is not None or torch.equal(out, clean))

"""The serving example's steps: pages that run out, and buffers that nothing fills twice."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_paged_planned import planned, prompts  # noqa: E402


def test_pages_that_run_out_are_an_error(l2):
    serving, layer = planned("bf16", n_pages=6)
    x = prompts(40, 30, 70)
    with pytest.raises(RuntimeError, match="status %d" % l2.paged.NO_ROOM):
        serving.serve_planned(layer, x, 3, 90)
    assert int(layer.free_count) == 6 and sorted(layer.free_pages.tolist()) == list(range(6)) and int(layer.lengths.abs().sum()) == 0 and bool((layer.table == -1).all())
    layer.status.zero_()
    outs, _, _ = serving.serve_planned(layer, x[:2], 3, 90)
    _, other = planned("bf16")
    assert all(torch.equal(a, b) for a, b in zip(outs, serving.serve_planned(other, x[:2], 3, 90)[0]))

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


def test_a_step_with_tables_of_the_host_fills_no_buffer(l2, monkeypatch):
    import paged_serving
    layer = paged_serving.PagedLayer(256, 4, 2, cache="f16", n_pages=8, page_size=16, positions=64)
    x, = prompts(40)
    sequence = {"length": 0, "table": []}

    def zeros(*args, **kw):
        raise AssertionError("every row is written anyway")

    monkeypatch.setattr(torch, "zeros", zeros)
    out = layer.step(x, [sequence], [40])
    assert out.isfinite().all() and int(layer.status) == 0

"""The paged serving example's pages: who has them, and what happens where there are none."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def layer_of(pages, **kw):
    import paged_serving
    return paged_serving, paged_serving.PagedLayer(256, 4, 2, cache="bf16", n_pages=pages, page_size=16, positions=512, **kw)


def prompts(*lengths):
    rng = np.random.default_rng(2)
    return [torch.from_numpy(rng.standard_normal((n, 256)).astype(np.float32)).cuda() * 0.05 for n in lengths]


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_pages_of_sequences_that_have_ended_come_back(window, sinks):
    serving, layer = layer_of(14, window=window, sinks=sinks)
    x = prompts(40, 70, 5, 33)  # 3 + 5 + 1 + 3 pages and one more each at most
    first, _, _ = serving.serve(layer, x, 4, 64)
    for _ in range(5):
        assert sorted(layer.free) == list(range(14))
        again, _, _ = serving.serve(layer, x, 4, 64)
        assert all(torch.equal(a, b) for a, b in zip(first, again))  # (whichever pages they got)
    assert int(layer.status) == 0


def test_a_step_without_room_changes_nothing():
    serving, layer = layer_of(6)
    a, b = ({"length": 0, "table": []} for _ in "ab")
    x, = prompts(120)
    layer.step(x[:50], [a, b], [20, 30])
    before = (dict(a, table=list(a["table"])), dict(b, table=list(b["table"])), list(layer.free))
    with pytest.raises(RuntimeError, match="5 pages needed, 2 left"):
        layer.step(x[50:], [a, b], [30, 40])
    assert (a, b, layer.free) == before
    layer.step(x[50:60], [a, b], [5, 5])
    assert a["length"] == 25 and b["length"] == 35 and len(layer.free) == 1
    layer.release(a), layer.release(b)
    assert sorted(layer.free) == list(range(6)) and not a["table"]

"""The paged serving example with tables on the device, and with a cache in 4 bits, against the same layer in 64 bits over whole sequences."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_paged_serving import whole  # noqa: E402


def prompts(*lengths, dim=256):
    rng = np.random.default_rng(3)
    return [torch.from_numpy(rng.standard_normal((n, dim)).astype(np.float32)).cuda() * 0.05 for n in lengths]


def planned(cache, n_pages=64, **kw):
    import paged_serving
    return paged_serving, paged_serving.PlannedLayer(256, 4, 2, cache=cache, n_pages=n_pages, page_size=16, positions=512, n_seqs=5, budget=90, **kw)


def check(layer, x, outs, bits, tokens, window, sinks):
    for p, out in zip(x, outs):
        own = [out[len(p) - 1 + i:len(p) + i] for i in range(tokens)]
        want = whole(layer, torch.cat([p] + [y / (y.square().mean() + 1e-5).sqrt() for y in own]), window, sinks)
        # K and V (and the queries) are rounded to `bits` and a sign; scores of a few units turn that into some times as much, relative to the rows' size
        assert float((out.double() - want).norm() / want.norm()) < 8 * 2.0 ** -(bits + 1)


# 4 bits: an element is off by half a step of a fifteenth of the row's range, five or six times its standard deviation
@pytest.mark.parametrize("cache,bits", [("f16", 10), ("i8", 6), ("u4", 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 3)])
def test_sequences_in_planned_steps_are_the_sequences_whole(l2, cache, bits, window, sinks):
    serving, layer = planned(cache, window=window, sinks=sinks)
    x = prompts(1, 130, 17, 64, 200)
    outs, steps, rows = serving.serve_planned(layer, x, 5, 90)
    assert int(layer.status) == 0 and rows == sum(len(p) + 5 for p in x) and steps >= 7
    check(layer, x, outs, bits, 5, window, sinks)
    # every page has come back, once
    assert int(layer.free_count) == 64 and sorted(layer.free_pages.tolist()) == list(range(64)) and int(layer.lengths.abs().sum()) == 0 and bool((layer.table == -1).all())
    again, _, _ = serving.serve_planned(layer, x, 5, 90)  # (whichever pages they get)
    assert all(torch.equal(a, b) for a, b in zip(outs, again)) and int(layer.status) == 0


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 3)])
def test_a_cache_in_4_bits_with_tables_of_the_host(l2, window, sinks):
    import paged_serving
    layer = paged_serving.PagedLayer(256, 4, 2, cache="u4", n_pages=64, page_size=16, positions=512, window=window, sinks=sinks)
    x = prompts(1, 130, 17, 64, 200)
    outs, _, rows = paged_serving.serve(layer, x, 5, 90)
    assert int(layer.status) == 0 and sorted(layer.free) == list(range(64))
    check(layer, x, outs, 3, 5, window, sinks)


def test_a_planned_step_without_room_brings_nothing(l2):
    serving, layer = planned("bf16", n_pages=6)
    x, = prompts(90)
    layer.step_planned(x[:50], [20, 30, 0, 0, 0])
    assert int(layer.status) == 0 and layer.lengths.tolist() == [20, 30, 0, 0, 0] and int(layer.free_count) == 2
    layer.step_planned(x, [40, 40, 10, 0, 0])
    assert int(layer.status) == l2.paged.NO_ROOM and layer.lengths.tolist() == [20, 30, 0, 0, 0] and int(layer.free_count) == 2
    layer.status.zero_()
    layer.end([1])
    layer.step_planned(x[:41], [30, 0, 11, 0, 0])
    assert int(layer.status) == 0 and layer.lengths.tolist() == [50, 0, 11, 0, 0] and int(layer.free_count) == 1


def test_several_steps_of_a_layer_in_a_graph(l2):
    """Plan, append, attention and the norms around it, captured once: a batch of single tokens that grows by itself."""
    torch.manual_seed(0)
    heads, kv_heads, n = 4, 2, 5
    shape = (40, 16, kv_heads, 64)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in "kv")
    pairs = [torch.zeros((40, kv_heads, 16, 2), dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    pages = l2.KvPages(k, v, *pairs)
    ints = lambda *s, fill=0: torch.full(s, fill, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lengths, start, status = ints(n, 8, fill=-1), ints(n), ints(n + 1), ints(1)
    tables = l2.KvTables(table, lengths, torch.arange(40, dtype=torch.int32, device="cuda"), ints(1, fill=40), 16, status=status)
    batch = l2.KvBatch(table, lengths, start, n, 1, status=status)
    one, weight = ints(n, fill=1), torch.rand(heads * 128, device="cuda") + 0.5
    stream, normed = torch.zeros((n, heads * 128), device="cuda"), torch.zeros((n, heads * 128), dtype=torch.bfloat16, device="cuda")
    new, out = torch.randn((2, n, kv_heads, 128), device="cuda"), torch.zeros((n, heads, 128), dtype=torch.bfloat16, device="cuda")
    work = torch.empty(pages.workspace_bytes(batch, heads), dtype=torch.uint8, device="cuda")

    def step():
        tables.plan(one, start, n, 1)
        pages.append(batch, new[0], new[1])
        l2.block_norm(None, stream, normed, pre_weight=weight)
        pages.attend(batch, normed.view(n, heads, 128), out, workspace=work)
        l2.block_norm(out.view(n, -1), stream, normed, residual_out=stream, post_weight=weight, pre_weight=weight, scale=0.5)

    begin = torch.randn((n, heads * 128), device="cuda")
    kept = []
    for captured in (False, True):
        tables.release(ints(n))
        stream.copy_(begin)
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step()
        for i in range(60):
            new.copy_(torch.sin(torch.arange(new.numel(), device="cuda").view(new.shape) * (1.0 + i)))
            graph.replay() if captured else step()
        kept.append((stream.clone(), normed.clone(), out.clone()))
        assert lengths.tolist() == [60] * n and int(status) == 0
    assert all(torch.equal(a, b) for a, b in zip(*kept)) and kept[0][0].isfinite().all()

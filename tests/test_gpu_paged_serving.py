"""The paged serving example: a layer over a paged cache against the same layer in 64 bits over whole sequences."""
import math

import numpy as np
import pytest

from conftest import dequant_dense

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def whole(layer, x, window, sinks):
    """The layer on a whole sequence at once, in 64 bits."""
    w = {n: torch.from_numpy(dequant_dense(*t, 64)).cuda() for n, t in layer.weights.items()}
    n, g = len(x), layer.heads // layer.kv_heads
    x = x.double()
    q, k, v = ((x @ w[i].T).view(n, -1, 128) for i in "qkv")
    cos, sin = (t[:n].double()[:, None] for t in layer.rope)

    def turn(t):
        a, b = t[..., :64], t[..., 64:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(g, 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(128)
    back = torch.arange(n, device="cuda")[:, None] - torch.arange(n, device="cuda")
    seen = back >= 0
    if window:
        seen &= (back < window) | (torch.arange(n, device="cuda") < sinks)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    return torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ w["o"].T


@pytest.mark.parametrize("cache,bits", [("f16", 10), ("bf16", 7), ("i8", 6)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 3)])
def test_sequences_in_steps_are_the_sequences_whole(l2, cache, bits, window, sinks):
    import paged_serving
    layer = paged_serving.PagedLayer(256, 4, 2, cache=cache, n_pages=64, page_size=16, positions=512, window=window, sinks=sinks)
    rng = np.random.default_rng(3)
    prompts = [torch.from_numpy(rng.standard_normal((n, 256)).astype(np.float32)).cuda() * 0.05 for n in (1, 130, 17, 64, 200)]
    outs, steps, rows = paged_serving.serve(layer, prompts, 5, 90)
    assert int(layer.status) == 0 and rows == sum(len(p) + 5 for p in prompts) and steps >= 7
    assert len(layer.free) >= 1 and len(set(layer.free)) == len(layer.free)
    for p, out in zip(prompts, outs):
        own = [out[len(p) - 1 + i:len(p) + i] for i in range(5)]
        x = torch.cat([p] + [y / (y.square().mean() + 1e-5).sqrt() for y in own])
        want = whole(layer, x, window, sinks)
        # K and V (and the queries) are rounded to `bits` and a sign; scores of a few units turn that into some times as much, relative to the rows' size
        assert float((out.double() - want).norm() / want.norm()) < 8 * 2.0 ** -(bits + 1)

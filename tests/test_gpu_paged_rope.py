"""RoPE of the paged cache against that of this library's models: the oracle's rope and attention, and l2_attention_decode_dev."""
import math

import numpy as np
import pytest

from test_gpu_attention import HS, oracle_attention, run_gpu

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from paged_reference import UNIT, Case  # noqa: E402
from test_gpu_paged import BF16, F16, F32, I8, rotate  # noqa: E402


def turned(orc, x, first, heads):
    """Rows [n, heads, 128] at positions first .. as orc_rope turns them (f32)."""
    import ctypes as C
    f = lambda a: a.ctypes.data_as(C.POINTER(C.c_float))
    out, spare = x.cpu().numpy().copy(), np.zeros((heads, HS), np.float32)
    for i in range(len(out)):
        row = np.ascontiguousarray(out[i])
        orc.lib().orc_rope(f(row), f(spare), first + i, heads, 0, HS)
        out[i] = row
    return torch.from_numpy(out)


# the appended key is the key that l2_attention_decode_dev appends, rounded to the cache's type; q likewise
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (32, 32)])
@pytest.mark.parametrize("cache", [F16, BF16, I8])
def test_keys_are_those_of_the_token_loop(l2, orc, cache, heads, kv_heads):
    rng = np.random.default_rng(heads)
    rope = l2.KvRope(1024)
    for pos in (0, 1, 2, 63, 300, 1023):
        q, k, v = (rng.standard_normal(n * HS).astype(np.float32) for n in (heads, kv_heads, kv_heads))
        empty = np.zeros((1024, kv_heads, HS), np.float32)
        _, keys, _ = run_gpu(l2, q, k, v, empty, empty.copy(), pos, heads, kv_heads, 1024)
        want = torch.from_numpy(keys[pos:pos + 1]).cuda()
        dq, dk, dv = (torch.from_numpy(t).cuda().view(1, -1, HS) for t in (q, k, v))
        c, plain = (Case([1], [pos + 1], kv_heads=kv_heads, group=heads // kv_heads, cache=cache) for _ in "ab")
        pages, batch = c.handles(l2)
        q_out = torch.empty((1, heads, HS), device="cuda")
        pages.append(batch, dk, dv, rope=rope, q=dq, q_out=q_out)
        pages, batch = plain.handles(l2)
        pages.append(batch, want, dv)  # the turned key as it is
        assert torch.equal(c.k, plain.k) and torch.equal(c.v, plain.v)
        if cache == I8:
            assert torch.equal(c.scales[0], plain.scales[0])
        exact = turned(orc, dq, pos, heads)
        assert ((q_out.cpu() - exact).abs() <= 1e-6 + 1e-6 * exact.abs()).all()
        # the tables' rotation is the default of the tables; another one has to be named
        pages, batch = plain.handles(l2)
        pages.append(batch, dk, dv, rope=tuple(rope), rotation="model", q=dq, q_out=(again := torch.empty_like(q_out)))
        assert torch.equal(again, q_out) and torch.equal(plain.k, c.k)
        pages.append(batch, dk, dv, rope=rope, rotation="pairs", q=dq, q_out=(pairs := torch.empty_like(q_out)))
        pages.append(batch, dk, dv, rope=tuple(rope), q=dq, q_out=again)
        assert torch.equal(again, pairs)
        want = rotate(dq, *rope, torch.tensor([pos]))
        assert ((pairs - want).abs() <= 3 * 2.0**-24 * 2 * float(want.abs().max())).all()
        assert pos == 0 or float((pairs - q_out).abs().max()) > 0.1


# one sequence, as one chunk and token by token, against l2_attention_decode_dev and the oracle
@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 1)])
def test_a_sequence_is_that_of_the_token_loop(l2, orc, cache, heads, kv_heads):
    n, group, u = 70, heads // kv_heads, UNIT[cache]
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal((n, h, HS)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
    dq, dk, dv = (torch.from_numpy(t).cuda() for t in (q, k, v))
    want = torch.empty((n, heads, HS), dtype=torch.float64)
    kc, vc = (np.zeros((n, kv_heads, HS), np.float32) for _ in "kv")
    for pos in range(n):
        mine, k1, v1 = run_gpu(l2, q[pos].ravel(), k[pos].ravel(), v[pos].ravel(), kc, vc, pos, heads, kv_heads, n)
        theirs, _, _ = oracle_attention(orc, q[pos].ravel(), k[pos].ravel(), v[pos].ravel(), kc, vc, pos, heads, kv_heads)
        assert (np.abs(mine - theirs) <= 1e-5 + 1e-4 * np.abs(theirs)).all()
        kc, vc = k1, v1
        want[pos] = torch.from_numpy(theirs).view(heads, HS)
    # q, k and v are rounded to u, and so are the probabilities: scores move by (2 u + u^2) sum |q| |k| scale, a probability by twice that in its exponent
    tq, tk = (turned(orc, t, 0, h).double() for t, h in ((dq, heads), (dk, kv_heads)))
    tk, tv = (t.repeat_interleave(group, 1) for t in (tk, torch.from_numpy(v).double()))
    seen = torch.ones((n, n), dtype=torch.bool).tril()
    p = torch.softmax((torch.einsum("ihd,jhd->hij", tq, tk) / math.sqrt(HS)).masked_fill(~seen, -math.inf), -1)
    move = (torch.einsum("ihd,jhd->hij", tq.abs(), tk.abs()) / math.sqrt(HS) * (2 * u + u * u) * seen).amax(-1)
    rel = torch.expm1(2 * move) + 2 * u + 2.0**-16 + 1e-4
    bound = torch.einsum("hij,jhd->ihd", p, tv.abs()) * rel.T[..., None] + 1e-5
    for steps in ([n], [33, 30, 1, 1, 5], [1] * n):
        c = Case([1], [n], kv_heads=kv_heads, group=group, cache=cache, page=16)
        out, at = torch.empty((n, heads, HS), device="cuda"), 0
        for r in steps:
            c.kv, c.rows, c.row_start, c.n = [at + r], [r], torch.tensor([0, r], dtype=torch.int32), r
            c.device_arrays()
            pages, batch = c.handles(l2)
            q16 = torch.empty((r, heads, HS), dtype=cache, device="cuda")
            pages.append(batch, dk[at:at + r], dv[at:at + r], rope=l2.KvRope(n), q=dq[at:at + r], q_out=q16)
            pages.attend(batch, q16, out[at:at + r])
            at += r
        err = (out.cpu().double() - want).abs()
        assert (err <= bound).all(), (steps[:3], float((err / bound).max()))


@pytest.mark.parametrize("cache,bits", [("f16", 10), ("bf16", 7), ("i8", 6)])
def test_the_serving_layer_as_the_token_loop(l2, cache, bits):
    import paged_serving
    layer = paged_serving.PagedLayer(256, 4, 2, cache=cache, n_pages=16, page_size=16, positions=128, rotation="model")
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((60, 256)).astype(np.float32)).cuda() * 0.05
    out, _, _ = paged_serving.serve(layer, [x], 0, 25)
    q, k, v = (layer._project(name, x).cpu().numpy() for name in "qkv")
    kc, vc = (np.zeros((60, 2, HS), np.float32) for _ in "kv")
    rows = torch.empty((60, 4 * HS), device="cuda")
    for pos in range(60):
        got, kc, vc = run_gpu(l2, q[pos], k[pos], v[pos], kc, vc, pos, 4, 2, 60)
        rows[pos] = torch.from_numpy(got).cuda()
    want = layer._project("o", rows)
    assert float((out[0] - want).norm() / want.norm()) < 8 * 2.0 ** -(bits + 1)


def test_rotations_that_are_none(l2):
    c = Case([1], [1], cache=F16)
    pages, batch = c.handles(l2)
    x = torch.zeros((1, 2, HS), device="cuda", dtype=F32)
    with pytest.raises(ValueError, match="rotation"):
        pages.append(batch, x, x, rope=l2.KvRope(4), rotation="halves")

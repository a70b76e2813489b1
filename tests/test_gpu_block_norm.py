"""Norms before and after a block against the same in 64 bits."""
import itertools

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
TINY = {F32: 2.0**-149, F16: 2.0**-25, BF16: 2.0**-134}


def make(rows, dim, block=BF16, residual=F32, out=BF16, post=True, pre=True, gate=None, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return {"block": (rand(rows, dim) * size).to(block) if block else None, "residual": (rand(rows, dim) * 3 * size).to(residual) if residual else None,
            "post_weight": 1 + 0.3 * rand(dim) if post else None, "pre_weight": 1 + 0.3 * rand(dim) if pre else None,
            "gate": None if gate is None else rand(dim).to(gate[1]) if gate[0] == "channel" else rand(rows, dim).to(gate[1])}


def want(a, scale, eps):
    """(r, out) in 64 bits and what each may be off by before it is rounded to its type: a product or sum is off by half a unit of f32, a sum of dim squares by (dim / 2 + 2)
    of them at most (a thread's elements one after the other, then pairs: 32 + 10 of them suffice), its root, inverse and products by a few more."""
    u, chain = 2.0**-24, 48
    r, slack = 0.0, 0.0
    if a["block"] is not None:
        t = a["block"].double()
        slack_t = torch.zeros_like(t)
        if a["post_weight"] is not None:
            t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * a["post_weight"].double()
            slack_t = (chain / 2 + 6) * u * t.abs()
        if a["gate"] is not None:
            g = a["gate"].double()
            t, slack_t = t * g, slack_t * g.abs() + 2 * u * (t * g).abs()
        r, slack = scale * t, abs(scale) * slack_t + 2 * u * abs(scale) * t.abs()
    if a["residual"] is not None:
        r = r + a["residual"].double()
    slack = slack + 2 * u * r.abs()
    f = 1 / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    w = a["pre_weight"].double() if a["pre_weight"] is not None else torch.ones((), dtype=torch.float64, device="cuda")
    # the row's factor moves with the elements: by the norm of their slack over the row's norm
    move = slack.square().sum(-1, keepdim=True).sqrt() / r.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-300)
    out = r * f * w
    return r, slack, out, (slack * f * w.abs()) + out.abs() * (move + (chain / 2 + 8) * u)


def check(got, exact, slack):
    t = got.dtype
    room = slack + UNIT[t] * (exact.abs() + slack) + TINY[t]
    bad = ~((got.double() - exact).abs() <= room)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), float(((got.double() - exact).abs() / room).max()))


def run(l2, a, out=BF16, residual_out=F32, scale=1.0, eps=1e-5):
    first = a["block"] if a["block"] is not None else a["residual"]
    o = torch.full(first.shape, 7.0, dtype=out, device="cuda") if out else None
    r = torch.full(first.shape, 7.0, dtype=residual_out, device="cuda") if residual_out else None
    l2.block_norm(a["block"], a["residual"], o, residual_out=r, post_weight=a["post_weight"], pre_weight=a["pre_weight"], gate=a["gate"], scale=scale, eps=eps)
    return r, o


def compare(l2, a, out=BF16, residual_out=F32, scale=1.0, eps=1e-5):
    r, o = run(l2, a, out, residual_out, scale, eps)
    er, sr, eo, so = want(a, scale, eps)
    if r is not None:
        check(r, er, sr)
    if o is not None:
        check(o, eo, so)


# every number of elements a thread, with whole fours and without; rows of a warp and of a CTA, more rows than CTAs
@pytest.mark.parametrize("rows", [1, 3, 700, 3000])
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 31, 64, 128, 130, 252, 256, 509, 512, 513, 1024, 1500, 4096, 5120, 8192])
def test_sizes(l2, rows, dim):
    compare(l2, make(rows, dim, gate=("channel", BF16)), scale=0.7)


@pytest.mark.parametrize("dim", [4097, 11008, 16384, 16388, 28672, 32767, 32768])
def test_long_rows(l2, dim):
    for rows in (2, 400):
        compare(l2, make(rows, dim), out=F32)


@pytest.mark.parametrize("block,residual", list(itertools.product([BF16, F16, F32], [BF16, F16, F32])))
@pytest.mark.parametrize("dim", [515, 640])
def test_types(l2, block, residual, dim):
    for out, gate in ((F16, ("element", F32)), (BF16, ("element", F16)), (F32, ("channel", BF16))):
        compare(l2, make(37, dim, block, residual, gate=gate), out=out, residual_out=residual, scale=-1.5)


def test_parts_that_are_absent(l2):
    for rows, dim in ((5, 640), (900, 130), (700, 640)):
        for post, pre, gate in itertools.product([True, False], [True, False], [None, ("channel", F32), ("element", BF16)]):
            compare(l2, make(rows, dim, post=post, pre=pre, gate=gate))
        compare(l2, make(rows, dim, residual=None, gate=("channel", F32)))
        compare(l2, make(rows, dim, block=None, post=False))           # the norm in front of a block alone
        compare(l2, make(rows, dim), out=None)                         # the residual stream alone
        compare(l2, make(rows, dim, post=False), out=None)
        compare(l2, make(rows, dim), residual_out=None)
        compare(l2, make(rows, dim, residual=None, post=False), residual_out=None)  # a plain norm


def test_in_place(l2):
    for rows, dim, t in ((5, 640, BF16), (700, 130, F32), (1000, 8192, BF16), (300, 32768, F32)):
        a = make(rows, dim, t, t, gate=("element", BF16))
        r, o = run(l2, a, out=t, residual_out=t, scale=0.5)
        block, residual = a["block"].clone(), a["residual"].clone()
        got = l2.block_norm(block, residual, block, residual_out=residual, post_weight=a["post_weight"], pre_weight=a["pre_weight"], gate=a["gate"], scale=0.5)
        assert got[0] is residual and got[1] is block and torch.equal(residual, r) and torch.equal(block, o)


def test_strides(l2):
    """Parts of larger arrays, starts on any boundary of elements, one row for all."""
    for start, gap in ((0, 0), (4, 8), (1, 0), (0, 3), (3, 5)):
        rows, dim = 50, 512
        a = make(rows, dim, gate=("element", BF16))
        plain = run(l2, a)

        def inside(t):
            room = torch.full((rows, start + dim + gap), 9.0, dtype=t.dtype, device="cuda")
            room[:, start:start + dim] = t
            return room, room[:, start:start + dim]

        b = {n: inside(a[n])[1] for n in ("block", "residual", "gate")}
        (ro, r), (oo, o) = (inside(torch.zeros_like(x)) for x in plain)
        l2.block_norm(b["block"], b["residual"], o, residual_out=r, post_weight=a["post_weight"], pre_weight=a["pre_weight"], gate=b["gate"])
        for got, exp, room in ((r, plain[0], ro), (o, plain[1], oo)):
            torch.testing.assert_close(got, exp, rtol=2.0**-7 if got.dtype == BF16 else 1e-5, atol=1e-6)
            room[:, start:start + dim] = 9.0
            assert (room == 9.0).all()
        one = {n: a[n][3:4].expand(rows, dim) for n in ("block", "residual", "gate")}
        same = run(l2, {**a, **one})
        assert all(torch.equal(x, x[:1].expand(rows, dim)) for x in same)
        check(same[0], *(x.expand(rows, dim) for x in want({**a, **{n: one[n][:1] for n in one}}, 1.0, 1e-5)[:2]))


@pytest.mark.parametrize("dim", [515, 640])
def test_values_at_the_edges(l2, dim):
    a = make(8, dim, F32, F32)
    a["block"][0], a["residual"][0] = 0, 0                       # 0 / sqrt(eps)
    a["block"][1], a["residual"][1] = 1e-30, 1e-30
    a["block"][2] *= 1e15
    a["residual"][3] *= 1e15
    compare(l2, a, out=F32)
    clean = run(l2, a, out=F32)
    for value in (float("nan"), float("inf")):                   # a row of it, and the others keep their bits
        b = {n: None if t is None else t.clone() for n, t in a.items()}
        b["block"][5, 7] = value
        b["residual"][6, 9] = value
        r, o = run(l2, b, out=F32)
        assert not r[5].isfinite().all() and not o[5].isfinite().all() and not o[6].isfinite().all()
        keep = [0, 1, 2, 3, 4, 7]
        assert torch.equal(r[keep], clean[0][keep]) and torch.equal(o[keep], clean[1][keep])
        assert torch.equal(r[6, :9], clean[0][6, :9])
    zero = make(3, dim, F32, F32)
    zero["block"].zero_(), zero["residual"].zero_()
    _, o = run(l2, zero, out=F32, eps=0.0)
    assert o.isnan().all()                                       # 0 / 0, as the formula says


def test_no_rows(l2):
    a = make(0, 640)
    r, o = run(l2, a)
    assert r.shape == (0, 640) and o.shape == (0, 640)


def test_refusals(l2):
    a = make(6, 640)
    out, r = torch.zeros((6, 640), dtype=BF16, device="cuda"), torch.zeros((6, 640), device="cuda")
    good = dict(block=a["block"], residual=a["residual"], out=out, residual_out=r, post_weight=a["post_weight"], pre_weight=a["pre_weight"])
    l2.block_norm(**good)
    room = torch.zeros((7, 640), device="cuda")
    wide = torch.zeros((6, 700), device="cuda")
    for bad in (dict(block=a["block"][:5]), dict(residual=a["residual"][:, :639]), dict(out=out.cpu()), dict(block=a["block"].T.contiguous().T), dict(post_weight=a["post_weight"].half()),
                dict(pre_weight=a["pre_weight"][:10]), dict(gate=torch.zeros(6, device="cuda")), dict(gate=torch.zeros(641, device="cuda")), dict(block=None, residual=None),
                dict(block=a["block"][0]), dict(post_weight=torch.zeros(1280, device="cuda")[::2])):
        with pytest.raises(ValueError):
            l2.block_norm(**{**good, **bad})
    for bad in (dict(block=a["block"].int()), dict(out=None, residual_out=None), dict(block=None), dict(eps=-1.0), dict(eps=float("nan")), dict(scale=float("inf")), dict(scale=float("nan")),
                dict(residual=room[:6], residual_out=room[1:]), dict(residual_out=a["residual"][:, :640].expand(6, 640)[:1].expand(6, 640)), dict(residual_out=wide[:, :640], out=wide[:, 30:670]),
                dict(residual_out=a["residual"], gate=a["residual"]), dict(out=a["residual"], residual_out=None), dict(out=out[:1].expand(6, 640)),
                dict(out=a["block"], residual=a["block"]), dict(residual_out=wide.view(-1)[:3840].view(6, 640), pre_weight=wide.view(-1)[100:740])):
        with pytest.raises(l2.L2Error):
            l2.block_norm(**{**good, **bad})
    with pytest.raises(l2.L2Error):
        big = torch.zeros((1, 32769), device="cuda")
        l2.block_norm(big, None, torch.zeros_like(big))


def test_in_a_graph_and_on_a_stream(l2):
    a = make(16, 4096)
    out, r = torch.zeros((16, 4096), dtype=BF16, device="cuda"), torch.zeros((16, 4096), device="cuda")
    call = lambda **kw: l2.block_norm(a["block"], a["residual"], out, residual_out=r, post_weight=a["post_weight"], pre_weight=a["pre_weight"], **kw)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    a["block"].normal_()
    graph.replay()
    er, sr, eo, so = want(a, 1.0, 1e-5)
    check(r, er, sr), check(out, eo, so)
    side = torch.cuda.Stream()
    a["block"].normal_()
    side.wait_stream(torch.cuda.current_stream())
    call(stream=side.cuda_stream)
    side.synchronize()
    er, sr, eo, so = want(a, 1.0, 1e-5)
    check(r, er, sr), check(out, eo, so)

"""Tables planned and taken back on the device against lists on the host."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


class Lists:
    """Who has which pages, as lists: what l2_kv_plan and l2_kv_release say they do, page by page."""

    def __init__(self, lengths, width, page, n_pages, seed=0):
        rng = np.random.default_rng(seed)
        order = rng.permutation(n_pages).tolist()
        self.page, self.width, self.n_pages = page, width, n_pages
        self.kv = list(lengths)
        self.table = []
        for n in lengths:
            used = -(-n // page)
            self.table.append([order.pop() for _ in range(used)] + [-1] * (width - used))
        self.free = order + [-5] * (n_pages - len(order))
        self.count = len(order)
        self.missed = False

    def device(self, l2):
        put = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
        self.d = {"table": put(self.table).reshape(len(self.kv), self.width), "kv": put(self.kv), "free": put(self.free), "count": put([self.count])}
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        return l2.KvTables(self.d["table"], self.d["kv"], self.d["free"], self.d["count"], self.page, status=self.status)

    def plan(self, new, n_rows, max_rows):
        """(row_start, slots, positions), or None without room."""
        new = [n if 0 <= n <= max_rows and 0 <= k and k + n <= self.width * self.page else 0 for n, k in zip(new, self.kv)]
        need = [-(-(k + n) // self.page) - -(-k // self.page) if n else 0 for n, k in zip(new, self.kv)]
        if sum(need) > self.count or sum(new) > n_rows:
            return None
        start, slots, positions = [0], [], []
        for b, n in enumerate(new):
            for j in range(self.kv[b], self.kv[b] + n):
                if j % self.page == 0:
                    self.count -= 1
                    self.table[b][j // self.page] = self.free[self.count]
                page = self.table[b][j // self.page]
                self.missed |= page < 0  # (cut back into a page that a window has given back)
                slots.append(page * self.page + j % self.page if page >= 0 else -1)
                positions.append(j)
            self.kv[b] += n
            start.append(start[-1] + n)
        pad = [-1] * (n_rows - len(slots))
        return start, slots + pad, positions + pad

    def release(self, keep=None, window=0, sinks=0):
        gone = []
        for b, n in enumerate(self.kv):
            k = n if keep is None else min(n, keep[b])
            entries = []
            if window:
                entries = [i for i in range(-(-k // self.page)) if i >= -(-sinks // self.page) and (i + 1) * self.page <= k - window + 1]
            entries += range(-(-k // self.page), -(-n // self.page))
            gone += [(b, i) for i in entries if self.table[b][i] >= 0]
            self.kv[b] = k
        for b, i in reversed(gone):
            self.free[self.count] = self.table[b][i]
            self.table[b][i] = -1
            self.count += 1

    def same(self):
        torch.cuda.synchronize()
        for name, want in (("table", self.table), ("kv", self.kv), ("count", [self.count])):
            assert self.d[name].cpu().numpy().reshape(-1).tolist() == np.array(want, np.int64).reshape(-1).tolist(), name
        assert self.d["free"][:self.count].tolist() == self.free[:self.count]
        owned = sorted([p for t in self.table for p in t if p >= 0] + self.free[:self.count])
        assert owned == list(range(self.n_pages))


def run_plan(tables, lists, new, n_rows, max_rows, slots=True, positions=True):
    row_start = torch.full((len(new) + 1,), 77, dtype=torch.int32, device="cuda")
    s = torch.full((n_rows,), 77, dtype=torch.int64, device="cuda") if slots else None
    p = torch.full((n_rows,), 77, dtype=torch.int32, device="cuda") if positions else None
    tables.plan(torch.tensor(new, dtype=torch.int32).cuda(), row_start, n_rows, max_rows, slots=s, positions=p)
    return row_start, s, p


def check_plan(tables, lists, new, n_rows, max_rows, **kw):
    row_start, s, p = run_plan(tables, lists, new, n_rows, max_rows, **kw)
    want = lists.plan(new, n_rows, max_rows)
    lists.same()
    assert want is not None
    assert row_start.tolist() == want[0] and (s is None or s.tolist() == want[1]) and (p is None or p.tolist() == want[2])
    return row_start


# one sequence, a few, more than a CTA has threads, more than one run of threads a CTA; steps of single tokens, chunks, and none
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("seqs", [1, 2, 31, 33, 64, 511, 513, 1500, 5000, 16384])
def test_steps(l2, seqs, page):
    rng = np.random.default_rng(seqs + page)
    width = 12
    lengths = rng.integers(0, width * page // 2, seqs).tolist()
    lengths[0] = 0
    lists = Lists(lengths, width, page, seqs * width + 3, seed=seqs)
    tables = lists.device(l2)
    for step in range(4):
        chunk = [1, 3, 2 * page + 1, 40][step]
        new = [int(n) for n in rng.choice([0, 1, 1, chunk], seqs)]
        new = [min(n, width * page - k) for n, k in zip(new, lists.kv)]
        check_plan(tables, lists, new, sum(new) + int(step % 2) * 37, max(new + [1]), slots=step != 2, positions=step != 3)
        if step == 1:  # some have ended, some lose a few rows
            keep = [int(rng.choice([0, max(0, k - 2), k, k + 5])) for k in lists.kv]
            tables.release(torch.tensor(keep, dtype=torch.int32).cuda())
            lists.release(keep)
            lists.same()
    tables.release(torch.zeros(seqs, dtype=torch.int32, device="cuda"))
    lists.release([0] * seqs)
    lists.same()
    assert lists.count == lists.n_pages and int(lists.status) == 0


def test_a_release_undoes_a_plan(l2):
    rng = np.random.default_rng(1)
    lists = Lists(rng.integers(0, 300, 200).tolist(), 64, 16, 200 * 64)
    tables = lists.device(l2)
    before = {n: t.clone() for n, t in lists.d.items()}
    for chunk in (1, 5, 400):
        run_plan(tables, lists, [int(x) for x in rng.integers(0, chunk + 1, 200)], 200 * chunk, chunk)
        tables.release(before["kv"])
        assert all(torch.equal(before[n], lists.d[n]) for n in before)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 1), (100, 16), (100, 17), (1000, 40), (5, 5000), (2**31 - 1, 2**31 - 1)])
def test_pages_behind_a_window(l2, window, sinks):
    rng = np.random.default_rng(2)
    lengths = [0, 1, 15, 16, 17, 100, 101, 2000, 999] + rng.integers(0, 2000, 60).tolist()
    lists = Lists(lengths, 130, 16, 130 * 69)
    tables = lists.device(l2)
    for step in range(5):
        new = [int(x) for x in rng.integers(0, 10, len(lengths))]
        check_plan(tables, lists, new, sum(new), 10)
        keep = [max(0, k - 3) for k in lists.kv] if step == 2 else None
        tables.release(torch.tensor(keep, dtype=torch.int32).cuda() if keep else None, window=window, sinks=sinks)
        lists.release(keep, window, sinks)
        lists.same()
    assert int(lists.status) == (l2.paged.BAD_PAGE if lists.missed else 0)


def test_a_whole_batch_in_one_step(l2):
    """Long prompts from nothing, thousands of pages each."""
    lists = Lists([0] * 5, 4000, 8, 20000)
    tables = lists.device(l2)
    new = [32000, 1, 0, 17, 31993]
    check_plan(tables, lists, new, sum(new), 32000)
    tables.release(torch.tensor([9, 0, 0, 17, 31000], dtype=torch.int32).cuda())
    lists.release([9, 0, 0, 17, 31000])
    lists.same()


def test_no_room(l2):
    """Too few pages or rows: nothing changes, nothing is brought, and it is said."""
    for n_pages, n_rows in ((7, 100), (40, 19)):
        lists = Lists([20, 16, 5], 8, 16, n_pages)
        tables = lists.device(l2)
        before = {n: t.clone() for n, t in lists.d.items()}
        row_start, s, p = run_plan(tables, lists, [10, 1, 60 if n_pages == 7 else 9], n_rows, 60)
        assert int(lists.status) == l2.paged.NO_ROOM and row_start.tolist() == [0] * 4 and (s == -1).all() and (p == -1).all()
        assert all(torch.equal(before[n], lists.d[n]) for n in before)
        lists.status.zero_()
        check_plan(tables, lists, [1, 1, 1], n_rows, 60)
        assert int(lists.status) == 0
    # exactly enough
    lists = Lists([16, 16], 8, 16, 4)
    check_plan(lists.device(l2), lists, [16, 1], 17, 16)
    assert lists.count == 0


def test_what_cannot_be_is_reported(l2):
    """Rows and lengths out of range: that sequence brings none and stays as it is; the others are planned."""
    for seqs in (6, 700):
        lists = Lists([10] * seqs, 4, 16, 4 * seqs)
        tables = lists.device(l2)
        lists.kv[1], lists.kv[3] = -1, 65
        lists.d["kv"].copy_(torch.tensor(lists.kv, dtype=torch.int32))
        new = [1] * seqs
        new[0], new[2], new[4] = -3, 9, 8
        row_start, s, p = run_plan(tables, lists, new, 10 * seqs, 8)
        want = lists.plan(new, 10 * seqs, 8)
        assert (row_start.tolist(), s.tolist(), p.tolist()) == (want[0], want[1], want[2])
        assert lists.d["kv"].tolist() == lists.kv and lists.d["table"].tolist() == lists.table
        assert int(lists.status) == l2.paged.BAD_ROWS | l2.paged.BAD_LENGTH
        lists.status.zero_()
        new = [0] * seqs
        new[5] = 2**31 - 1  # beyond the table, and beyond 31 bits together with the length
        run_plan(tables, lists, new, 10, 2**31 - 1)
        assert int(lists.status) == l2.paged.BAD_LENGTH and lists.d["kv"].tolist() == lists.kv
        # lengths to keep below zero, lengths that cannot be
        lists.status.zero_()
        keep = [5] * seqs
        keep[0] = -1
        tables.release(torch.tensor(keep, dtype=torch.int32).cuda())
        assert int(lists.status) == l2.paged.BAD_LENGTH
        assert lists.d["kv"].tolist()[:4] == [10, -1, 5, 65]


def test_entries_that_are_no_pages(l2):
    lists = Lists([40, 40], 8, 16, 16)
    tables = lists.device(l2)
    # a number in the free list that is none
    lists.d["free"][lists.count - 1] = 16
    row_start, s, _ = run_plan(tables, lists, [10, 10], 20, 10)
    assert int(lists.status) == l2.paged.BAD_PAGE and lists.d["table"][0, 3] == -1 and lists.d["table"][1, 3] == lists.free[lists.count - 2]
    assert s.tolist()[:8] == [lists.table[0][2] * 16 + i for i in range(8, 16)] and s.tolist()[8:10] == [-1, -1]
    # one in a table: stays there; -1 is none that is missed
    lists.status.zero_()
    lists.d["table"][1, 0] = -9
    lists.d["table"][1, 1] = -1
    tables.release(torch.tensor([50, 0], dtype=torch.int32).cuda())
    assert int(lists.status) == l2.paged.BAD_PAGE and lists.d["table"][1].tolist() == [-1 - 8, -1, -1, -1, -1, -1, -1, -1]
    # the number of free pages
    for wrong, nearest in ((-4, 0), (99, 16)):
        lists = Lists([40, 40], 8, 16, 16)
        tables = lists.device(l2)
        lists.d["count"].fill_(wrong)
        run_plan(tables, lists, [1, 1], 2, 1)
        assert int(lists.status) == l2.paged.BAD_PAGE and int(lists.d["count"]) == nearest
    # more pages given back than there are
    lists = Lists([40, 40], 8, 16, 16)
    tables = lists.device(l2)
    lists.d["count"].fill_(13)
    tables.release(torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert int(lists.status) == l2.paged.BAD_PAGE and int(lists.d["count"]) == 16 and lists.d["kv"].tolist() == [0, 0]


def test_no_sequences_and_no_rows(l2):
    lists = Lists([], 4, 16, 3)
    tables = lists.device(l2)
    row_start, s, p = run_plan(tables, lists, [], 5, 1)
    assert row_start.tolist() == [0] and (s == -1).all() and (p == -1).all() and int(lists.status) == 0
    tables.release()
    lists = Lists([5, 0], 4, 16, 3)
    tables = lists.device(l2)
    check_plan(tables, lists, [0, 0], 0, 0)
    assert int(lists.status) == 0


def test_refusals(l2):
    lists = Lists([5, 6], 4, 16, 9)
    tables = lists.device(l2)
    d = lists.d
    new, start = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        l2.KvTables(d["table"], d["kv"][:1], d["free"], d["count"], 16)
    with pytest.raises(ValueError):
        l2.KvTables(d["table"].long(), d["kv"], d["free"], d["count"], 16)
    with pytest.raises(ValueError):
        l2.KvTables(d["table"].cpu(), d["kv"], d["free"], d["count"], 16)
    with pytest.raises(ValueError):
        l2.KvTables(d["table"], d["kv"], d["free"], d["count"], 1 << 40)
    for bad in (dict(new_rows=new[:1]), dict(row_start=start[:2]), dict(slots=start), dict(positions=torch.zeros(5, dtype=torch.int32, device="cuda")), dict(n_rows=1 << 40), dict(new_rows=new.cpu())):
        with pytest.raises(ValueError):
            tables.plan(**{**dict(new_rows=new, row_start=start, n_rows=4, max_rows=4), **bad})
    for bad in (dict(n_rows=-1), dict(max_rows=-1)):
        with pytest.raises(l2.L2Error):
            tables.plan(**{**dict(new_rows=new, row_start=start, n_rows=4, max_rows=4), **bad})
    with pytest.raises(l2.L2Error):
        l2.KvTables(d["table"], d["kv"], d["free"], d["count"], 24).release()
    for bad in (dict(window=-1), dict(sinks=-1)):
        with pytest.raises(l2.L2Error):
            tables.release(**bad)
    with pytest.raises(ValueError):
        tables.release(window=1 << 40)
    lists.same()


def test_in_a_graph(l2):
    """A step's plan captured once: replays go on from where the tables are."""
    lists = Lists([3, 60, 0, 17], 40, 16, 160)
    tables = lists.device(l2)
    new = torch.zeros(4, dtype=torch.int32, device="cuda")
    keep = torch.zeros(4, dtype=torch.int32, device="cuda")
    start, slots = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(64, dtype=torch.int64, device="cuda")
    step = lambda: (tables.release(keep), tables.plan(new, start, 64, 40, slots=slots))  # noqa: E731
    keep.fill_(1 << 20)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    rng = np.random.default_rng(0)
    for _ in range(6):
        rows = [int(x) for x in rng.integers(0, 16, 4)]
        kept = [int(rng.choice([0, k, k, max(0, k - 1)])) for k in lists.kv]
        new.copy_(torch.tensor(rows, dtype=torch.int32)), keep.copy_(torch.tensor(kept, dtype=torch.int32))
        graph.replay()
        lists.release(kept)
        want = lists.plan(rows, 64, 40)
        lists.same()
        assert start.tolist() == want[0] and slots.tolist() == want[1]
    assert int(lists.status) == 0


def test_a_planned_step_through_the_cache(l2):
    """Plan, append, attend and release of several steps on the planned arrays, against the same with arrays of the host."""
    torch.manual_seed(0)
    for cache in ("u4", "i8", "bf16"):
        pools = []
        for _ in range(2):
            shape = (64, 16, 2, 64 if cache == "u4" else 128)
            k, v = (torch.zeros(shape, dtype={"u4": torch.uint8, "i8": torch.int8, "bf16": torch.bfloat16}[cache], device="cuda") for _ in "kv")
            scales = [] if cache == "bf16" else [torch.zeros((64, 2, 16, 2), dtype=torch.bfloat16, device="cuda") if cache == "u4" else torch.zeros((64, 2, 16), device="cuda") for _ in "kv"]
            pools.append(l2.KvPages(k, v, *scales))
        lists = Lists([0] * 3, 16, 16, 64)
        tables = lists.device(l2)
        start = torch.zeros(4, dtype=torch.int32, device="cuda")
        n = 70
        planned = l2.KvBatch(lists.d["table"], lists.d["kv"], start, n, 60, status=lists.status)
        for rows in ([30, 0, 12], [1, 40, 1], [1, 1, 1], [60, 1, 1]):
            new, q = torch.randn((2, n, 2, 128), device="cuda"), torch.randn((n, 8, 128), device="cuda").to(torch.bfloat16)
            tables.plan(torch.tensor(rows, dtype=torch.int32).cuda(), start, n, 60)
            pools[0].append(planned, new[0], new[1])
            out = pools[0].attend(planned, q, torch.zeros_like(q))
            lists.plan(rows, n, 60)
            host = l2.KvBatch(torch.tensor(lists.table, dtype=torch.int32).cuda(), torch.tensor(lists.kv, dtype=torch.int32).cuda(),
                              torch.tensor([0, *np.cumsum(rows)], dtype=torch.int32).cuda(), n, 60)
            pools[1].append(host, new[0], new[1])
            assert torch.equal(out, pools[1].attend(host, q, torch.zeros_like(q)))
            lists.same()
        assert int(lists.status) == 0

"""Pages kept on the device against the same bookkeeping on the host: whole numbers, equal."""
import random

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device=_dev())


def places(length, grids):
    """(time, height, width) of the first `length` tokens of a sequence."""
    out, at = [], 0
    grids = [g for g in grids if min(g[1:]) > 0]
    while len(out) < length:
        if grids and grids[0][0] == len(out):
            _, t, h, w = grids.pop(0)
            out += [(at + r // (h * w), at + r // w % h, at + r % w) for r in range(min(t * h * w, length))]
            at += max(t, h, w)
        else:
            out.append((at,) * 3)
            at += 1
    return out[:length]


class Host:
    """The definition, on the host, beside a state on the GPU."""

    def __init__(self, pages, sequences, columns, page):
        from w4a8_b200 import kvcache
        self.S, self.cols = page, columns
        self.free = list(range(pages))[::-1]
        self.held, self.len = [[] for _ in range(sequences)], [0] * sequences
        self.state = kvcache.PageState.empty(pages, sequences, columns, page, _dev())

    def plan(self, rows, counts, tokens=None, axes=1, grids=None):
        from w4a8_b200 import kvcache
        images, total = None, sum(counts)
        tokens = total if tokens is None else tokens
        if grids is not None:
            cu = [0]
            for g in grids:
                cu.append(cu[-1] + len(g))
            images = (_i(cu), _i([s for g in grids for s in g]).view(-1, 4))
        m = kvcache.pages_plan(self.state, _i(rows), _i(counts), tokens, axes=axes, images=images)
        table, lens, cu, slots, pos = [], [], [0], [], []
        for j, (r, n) in enumerate(zip(rows, counts)):
            was = self.len[r]
            while len(self.held[r]) * self.S < was + n:
                self.held[r].append(self.free.pop())
            self.len[r] += n
            table.append(self.held[r] + [-1] * (self.cols - len(self.held[r])))
            lens.append(was + n)
            cu.append(cu[-1] + n)
            slots += [self.held[r][p // self.S] * self.S + p % self.S for p in range(was, was + n)]
            pos += places(was + n, grids[j] if grids else [])[was:]
        assert m.page_table.tolist() == table and m.kv_lens.tolist() == lens and m.cu.tolist() == cu
        assert m.slots.tolist() == slots + [-1] * (tokens - total)
        for a in range(axes):
            assert m.positions[a].tolist() == [p[min(a, 2)] for p in pos] + [0] * (tokens - total)
        self.same()
        return m

    def shrink(self, rows, keep=None):
        from w4a8_b200 import kvcache
        kvcache.pages_shrink(self.state, _i(rows), None if keep is None else _i(keep))
        for r, n in list(zip(rows, keep or [0] * len(rows)))[::-1]:
            while len(self.held[r]) > -(-n // self.S):
                self.free.append(self.held[r].pop())
            self.len[r] = n
        self.same()

    def same(self):
        s = self.state
        assert s.status() == 0 and s.control.tolist() == [0] * 4
        assert s.free_pages.item() == len(self.free) and s.free[:len(self.free)].tolist() == self.free
        assert s.lens.tolist() == self.len
        assert s.table.tolist() == [h + [-1] * (self.cols - len(h)) for h in self.held]


@pytest.mark.parametrize("page,sequences,columns,seed", [(16, 1, 4, 0), (16, 9, 33, 1), (32, 40, 7, 2), (128, 300, 3, 3), (64, 17, 130, 4)])
def test_steps(page, sequences, columns, seed):
    r = random.Random(seed)
    h = Host(sequences * columns * 3 // 4 + 1, sequences, columns, page)
    for _ in range(12):
        rows = r.sample(range(sequences), r.randint(1, sequences))
        counts, left = [], len(h.free)
        for x in rows:
            most = min(columns * page - h.len[x], left * page)
            n = r.choice((0, 1, 2, page, r.randint(0, 3 * page), most))
            n = min(n, most)
            left -= -(-(h.len[x] + n) // page) - len(h.held[x])
            if left < 0:
                left += -(-(h.len[x] + n) // page) - len(h.held[x])
                n = 0
            counts.append(n)
        h.plan(rows, counts, tokens=sum(counts) + r.choice((0, 0, 5)), axes=r.choice((1, 2, 3, 4)))
        rows = r.sample(range(sequences), r.randint(1, sequences))
        if r.random() < 0.4:
            h.shrink(rows)
        else:
            h.shrink(rows, [r.randint(0, h.len[x]) for x in rows])


def test_a_shrink_undoes_a_plan():
    h = Host(60, 5, 20, 16)
    h.plan([0, 1, 2, 3, 4], [17, 1, 16, 0, 40])
    free, held, lens = list(h.free), [list(x) for x in h.held], list(h.len)
    h.plan([4, 2, 0], [100, 30, 9])
    h.shrink([4, 2, 0], [40, 16, 17])
    assert (h.free, h.held, h.len) == (free, held, lens)


def test_images():
    r = random.Random(5)
    h = Host(4000, 6, 600, 16)
    grids = []
    for s in range(6):
        g, at = [], r.randint(0, 3)
        for _ in range(s):
            g.append((at, r.choice((1, 1, 3)), r.randint(1, 9), r.randint(1, 9)))
            at += g[-1][1] * g[-1][2] * g[-1][3] + r.randint(0, 4)
        grids.append(g)
    grids[2].insert(1, (grids[2][0][0] + 1, 0, 5, 5))                     # holds nothing
    grids[5].append((1 << 30, 1 << 20, 1 << 20, 1 << 20))                 # not reached
    for counts in ([5, 1, 40, 0, 200, 300], [1] * 6, [0, 300, 0, 7, 800, 16], [2, 0, 0, 1, 3, 1]):
        h.plan(list(range(6)), counts, axes=3, grids=grids)
    h.plan([3, 1], [4, 4], axes=3, grids=[grids[3], grids[1]], tokens=20)
    h.plan([3, 1], [4, 4], axes=3, grids=[[], []])


def test_the_largest_batch_and_table():
    r = random.Random(6)
    h = Host(2048 * 4 + 70000, 2100, 40, 128)
    rows = r.sample(range(2100), 2048)
    h.plan(rows, [r.randint(0, 400) for _ in rows], axes=1)
    h.plan(rows[::-1], [1] * 2048, axes=3)
    h.shrink(rows, [h.len[x] // 2 for x in rows])
    big = Host(66000, 65536, 2, 16)
    big.plan([65535, 0, 32768, 31], [17, 32, 1, 5])
    big.shrink([0, 65535])
    long = Host(70000, 2, 66000, 16)
    long.plan([1, 0], [1000000, 3])
    long.plan([1], [1])
    long.shrink([1], [16])


def test_lengths_at_the_end_of_32_bits():
    """A sequence of just below 2^31 tokens: lengths, slots and positions at the end of the range."""
    from w4a8_b200 import kvcache
    dev, S = _dev(), 128
    cols = (2 ** 31 - 1) // S
    table = torch.full((1, cols), 7, dtype=torch.int32, device=dev)
    free = torch.tensor([3, cols - 1], dtype=torch.int32, device=dev)
    pages = torch.zeros(cols, dtype=torch.int32, device=dev)
    pages[:2] = free
    st = kvcache.PageState(pages, _i([2]), table, _i([(cols - 1) * S - 1]), S)
    m = kvcache.pages_plan(st, _i([0]), _i([S]), S, axes=2)
    assert m.kv_lens.tolist() == [cols * S - 1]
    assert m.slots.tolist() == [7 * S + S - 1] + [(cols - 1) * S + j for j in range(S - 1)]
    assert m.positions[1].tolist() == [(cols - 1) * S - 1 + j for j in range(S)]
    assert st.status() == 0
    kvcache.pages_plan(st, _i([0]), _i([2]), 2)
    assert st.status() == 16


REFUSED = [
    # rows, counts, tokens, reason
    ([0, 0], [1, 1], 2, 1), ([3], [1], 1, 1), ([-1], [1], 1, 1), ([0, 1], [1, -1], 4, 2), ([0, 1], [5, 6], 10, 4), ([0, 1], [1, 200], 201, 16),
    ([0, 1, 2], [60, 60, 60], 180, 16),                                   # 17 + 60 tokens, 64 fit 4 columns
    ([0, 1, 2], [40, 64, 50], 154, 8),                                    # 2 + 4 + 3 pages, 6 are free
    ([2 ** 31 - 1], [1], 1, 1), ([0], [2 ** 31 - 1], 5, 4), ([1, 2, 1], [0, 0, 0], 3, 1),
]


@pytest.mark.parametrize("rows,counts,tokens,why", REFUSED)
def test_refused_steps_change_nothing(rows, counts, tokens, why):
    from w4a8_b200 import kvcache
    h = Host(9, 3, 4, 16)
    h.plan([2, 0], [5, 17])
    m = kvcache.pages_plan(h.state, _i(rows), _i(counts), tokens, axes=2)
    assert h.state.status(reset=False) == why
    with pytest.raises(RuntimeError, match="pages: "):
        h.state.check()
    assert (m.page_table == -1).all() and (m.slots == -1).all()
    assert not m.kv_lens.any() and not m.cu.any() and not m.positions.any()
    h.same()
    h.plan([1, 2], [3, 20])


def test_refused_shrinks_change_nothing():
    from w4a8_b200 import kvcache
    h = Host(9, 3, 4, 16)
    h.plan([2, 0], [5, 17])
    for rows, keep, why in (([2], [6], 2), ([0, 0], [1, 1], 1), ([0], [-1], 2), ([3], None, 1), ([-1], None, 1)):
        kvcache.pages_shrink(h.state, _i(rows), None if keep is None else _i(keep))
        assert h.state.status() == why
        h.same()
    h.state.free_pages.fill_(9)                                           # more free than the stack has room for
    kvcache.pages_shrink(h.state, _i([0]))
    assert h.state.status() == 32
    h.state.free_pages.fill_(-1)
    kvcache.pages_plan(h.state, _i([1]), _i([1]), 1)
    assert h.state.status() == 32


def test_captured_steps_and_many_in_a_row():
    from w4a8_b200 import kvcache
    h, g = Host(300, 8, 30, 16), Host(300, 8, 30, 16)
    rows, counts = _i(list(range(8))), _i([3] * 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m = kvcache.pages_plan(g.state, rows, counts, 24, axes=3)
        kvcache.pages_shrink(g.state, rows[2:4])
    for step in range(12):
        graph.replay()
        want = h.plan(list(range(8)), [3] * 8, axes=3)
        h.shrink([2, 3])
        assert all(torch.equal(x, y) for x, y in zip(m, want))
        for a, b in ((g.state.free_pages, h.state.free_pages), (g.state.table, h.state.table), (g.state.lens, h.state.lens)):
            assert torch.equal(a, b)
    assert g.state.status() == 0


def test_refusals():
    from w4a8_b200 import kvcache
    dev = _dev()
    st = kvcache.PageState.empty(10, 3, 4, 16, dev)
    r, c = _i([0, 1]), _i([1, 1])
    seg = (_i([0, 1, 1]), _i([[0, 1, 1, 1]]))
    empty = kvcache.PageState.empty
    bad = [
        lambda: empty(0, 3, 4), lambda: empty(10, 0, 4), lambda: empty(10, 3, 0), lambda: empty(10, 3, 4, 24), lambda: empty(10, 65537, 1),
        lambda: empty(2 ** 27, 1, 1, 16), lambda: empty(10, 3, 4, 16, "cpu"),
        lambda: kvcache.PageState(st.free, st.free_pages, st.table, st.lens[:2], 16),
        lambda: kvcache.PageState(st.free.long(), st.free_pages, st.table, st.lens, 16),
        lambda: kvcache.PageState(st.free, st.free_pages, st.table.T, st.lens, 16),
        lambda: kvcache.pages_plan(st, r, c[:1], 2), lambda: kvcache.pages_plan(st, r.long(), c, 2), lambda: kvcache.pages_plan(st, r, c.cpu(), 2),
        lambda: kvcache.pages_plan(st, r, c, -1), lambda: kvcache.pages_plan(st, r, c, 2, axes=0), lambda: kvcache.pages_plan(st, r, c, 2, axes=5),
        lambda: kvcache.pages_plan(st, r, c, 2, images=seg), lambda: kvcache.pages_plan(st, r, c, 2, axes=3, images=(seg[0][:2], seg[1])),
        lambda: kvcache.pages_plan(st, r, c, 2, axes=3, images=(seg[0], seg[1][:, :3])),
        lambda: kvcache.pages_plan(st, _i([0] * 2049), _i([0] * 2049), 2), lambda: kvcache.pages_shrink(st, r, c[:1]),
        lambda: kvcache.pages_shrink(st, r.view(1, 2)),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    m = kvcache.pages_plan(st, r[:0], c[:0], 3)
    assert m.cu.tolist() == [0] and m.slots.tolist() == [-1] * 3 and m.page_table.shape == (0, 4)
    kvcache.pages_shrink(st, r[:0])
    kvcache.pages_plan(st, r, c, 2, axes=3, images=(_i([0, 0, 0]), seg[1][:0]))
    assert st.status() == 0 and st.lens.tolist() == [1, 1, 0]

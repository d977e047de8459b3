"""Block tables and slot maps against a plan made one entry after another."""
import numpy as np
import pytest

from _pages import i32
from bmo_jetson_amd import KVPages, RingError

pytestmark = pytest.mark.gpu

UNTOUCHED = -12345


class Model:
    """The plan as a loop over the entries, in Python's whole numbers."""

    def __init__(self, n_pages, page, n, width):
        self.n_pages, self.page, self.width = n_pages, page, width
        self.free = list(range(n_pages - 1, -1, -1))
        self.lens = [0] * n
        self.table = [[UNTOUCHED] * width for _ in range(n)]

    def plan(self, n_new, max_tok):
        P, pages = self.page, lambda x: -(-x // self.page)
        start, status, tok, wanted, given, back = 0, [], [], 0, 0, []
        starts, free = [], list(self.free)
        for b, n in enumerate(n_new):
            starts.append(start)
            length = self.lens[b]
            new = max(0, length + n)
            start += max(n, 0)
            state = 0
            if length < 0 or length > self.width * P or new > self.width * P or (n > 0 and start > max_tok):
                state = 2
            elif n > 0:
                need = pages(new) - pages(length)
                wanted += need
                if need and wanted > len(free):
                    state = 1
                else:
                    for j in range(need):
                        self.table[b][pages(length) + j] = free[len(free) - 1 - given - j]
                    given += need
            elif n < 0:
                back += [self.table[b][c] for c in range(pages(new), pages(length))]
            if n > 0:
                for i in range(n):
                    if len(tok) < max_tok:
                        pos = length + i
                        tok.append((self.table[b][pos // P] * P + pos % P, pos, b) if state == 0 else (-1, -1, b))
            if state == 0:
                self.lens[b] = new
            status.append(state)
        self.free = free[:len(free) - given] + back[::-1]
        return starts + [start], status, tok


def _device(gpu, pages, n, width):
    free = i32(gpu, np.full(pages.n_pages + 2, 5))
    pages.list_init(free, stream=gpu.cuda.current_stream())
    return free, i32(gpu, np.zeros(n)), i32(gpu, np.full((n, width), UNTOUCHED))


def _compare(m, free, lens, table):
    f = free.cpu().numpy()
    assert f[0] == len(m.free) and f[1] == 0
    assert f[2:2 + f[0]].tolist() == m.free
    assert lens.cpu().tolist() == m.lens
    assert table.cpu().tolist() == m.table


@pytest.mark.parametrize("n,page,n_pages,width,most,cap", [
    (1, 32, 4, 4, 40, 64), (7, 64, 30, 12, 200, 600), (64, 32, 100, 9, 40, 900), (300, 64, 400, 5, 90, 20000),
    (1024, 128, 900, 3, 100, 70000), (1500, 32, 2500, 6, 60, 60000), (2500, 64, 5000, 40, 1500, 900000)])
def test_plans_follow_one_another(gpu, n, page, n_pages, width, most, cap):
    pages = KVPages(1, n_pages, page, 1, 64)
    m = Model(n_pages, page, n, width)
    free, lens, table = _device(gpu, pages, n, width)
    r = np.random.default_rng(n)
    seen = set()
    for step in range(8):
        kind = r.integers(0, 10, n)
        n_new = np.where(kind < 5, r.integers(0, most, n), np.where(kind < 7, 1, -r.integers(0, most, n)))
        if step == 3:
            n_new = np.where(kind < 8, -2**31 + 1, n_new)  # most requests end
        if step == 6:
            n_new = np.ones(n, dtype=np.int64)
        out = [i32(gpu, np.full(size, UNTOUCHED)) for size in (n + 1, cap, cap, cap, n)]
        pages.plan(free, i32(gpu, n_new), lens, table, *out, stream=gpu.cuda.current_stream())
        start, status, tok = m.plan([int(x) for x in n_new], cap)
        seen |= set(status)
        assert out[0].cpu().tolist() == start and out[4].cpu().tolist() == status
        got = np.stack([x.cpu().numpy() for x in out[1:4]], axis=1)
        assert got[:len(tok)].tolist() == [list(t) for t in tok]
        assert (got[len(tok):] == UNTOUCHED).all()  # what lies behind the last token
        _compare(m, free, lens, table)
    assert seen == ({0} if n <= 64 else {0, 1} if n <= 1500 else {0, 1, 2})
    pages.close()


def test_a_growth_taken_back_restores_the_list(gpu):
    n, page, width = 40, 64, 20
    pages = KVPages(1, 300, page, 1, 128)
    m = Model(300, page, n, width)
    free, lens, table = _device(gpu, pages, n, width)
    first = np.arange(n) * 7
    pages.plan(free, i32(gpu, first), lens, table, slots=i32(gpu, np.zeros(first.sum())))
    m.plan(first.tolist(), int(first.sum()))
    before = free.clone(), lens.clone()
    grow = np.arange(n)[::-1] * 5
    pages.plan(free, i32(gpu, grow), lens, table, slots=i32(gpu, np.zeros(grow.sum())))
    m.plan(grow.tolist(), int(grow.sum()))
    _compare(m, free, lens, table)
    pages.plan(free, i32(gpu, -grow), lens, table)  # no outputs asked for
    assert gpu.equal(free, before[0]) and gpu.equal(lens, before[1])
    pages.close()


def test_lengths_and_requests_out_of_range(gpu):
    pages = KVPages(1, 50, 32, 1, 64)
    free, lens, table = _device(gpu, pages, 6, 4)
    lens.copy_(i32(gpu, [0, -3, 129, 128, 2**31 - 1, 0]))
    n_new = i32(gpu, [129, 1, 1, 1, 1, 128])
    out = [i32(gpu, np.full(size, UNTOUCHED)) for size in (7, 400, 400, 400, 6)]
    pages.plan(free, n_new, lens, table, *out)
    assert out[4].cpu().tolist() == [2, 2, 2, 2, 2, 0]
    assert lens.cpu().tolist() == [0, -3, 129, 128, 2**31 - 1, 128]
    slots = out[1].cpu().numpy()
    assert (slots[:133] == -1).all() and slots[133:261].tolist() == list(range(128)) and (slots[261:] == UNTOUCHED).all()
    assert int(free[0]) == 46
    # more tokens asked for than the arrays hold
    pages.plan(free, i32(gpu, [5, 2**31 - 1, 2**31 - 1, 2**31 - 1, 2**31 - 1, 0]), lens, table, *out)
    assert out[4].cpu().tolist() == [0, 2, 2, 2, 2, 0]
    assert lens.cpu().tolist()[0] == 5 and int(free[0]) == 45
    pages.close()


@pytest.mark.parametrize("n,width,n_pages", [(30, 10, 120), (2400, 4, 3500)])  # one workgroup, several
def test_replayed_from_a_graph(gpu, n, width, n_pages):
    """A captured step: every replay grows the entries from where the last one
    left them, with eager plans of the program's own in between."""
    page = 32
    pages = KVPages(1, n_pages, page, 1, 64)
    m = Model(n_pages, page, n, width)
    free, lens, table = _device(gpu, pages, n, width)
    ones, drop = np.arange(n) % 3, np.where(np.arange(n) % 4 == 0, -1, 0)
    a, c = i32(gpu, ones), i32(gpu, drop)
    cap = int(ones.sum())
    out = [i32(gpu, np.zeros(size)) for size in (n + 1, cap, cap, cap, n)]
    graph = gpu.cuda.CUDAGraph()
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side), gpu.cuda.graph(graph, stream=side):
        pages.plan(free, a, lens, table, *out, stream=gpu.cuda.current_stream())
        pages.plan(free, c, lens, table, stream=gpu.cuda.current_stream())
    gpu.cuda.current_stream().wait_stream(side)
    for step in range(25):
        graph.replay()
        start, status, tok = m.plan(ones.tolist(), cap)
        m.plan(drop.tolist(), 0)
        gpu.cuda.synchronize()
        assert out[1].cpu().tolist() == [t[0] for t in tok] and out[4].cpu().tolist() == status
        _compare(m, free, lens, table)
        if step % 6 == 5:
            end = np.where(np.arange(n) % 5 == step % 5, -10**6, 0)
            pages.plan(free, i32(gpu, end), lens, table, stream=gpu.cuda.current_stream())
            m.plan(end.tolist(), 0)
    pages.close()


def test_refusals(gpu):
    pages = KVPages(1, 8, 64, 1, 64)
    free, lens, table = _device(gpu, pages, 3, 4)
    with pytest.raises(ValueError):
        pages.plan(free[:-1], lens, lens, table)
    with pytest.raises(ValueError):
        pages.plan(free, lens[:2], lens, table)
    with pytest.raises(ValueError):
        pages.plan(free, lens, lens, table, slots=i32(gpu, [0]), positions=i32(gpu, [0, 1]))
    with pytest.raises(ValueError):
        pages.plan(free, lens, lens, table.t())
    from bmo_jetson_amd import lib
    L, P = lib(), lambda t: t.data_ptr()
    for n_batch, width in ((0, 4), (-1, 4), (3, 0), (3, (1 << 30) // 64 + 1)):
        assert L.bmo_kv_pages_plan(pages.handle, P(free), n_batch, P(lens), P(lens), P(table), width, None, 0, None, None,
                                   None, None, None) == 2
    assert L.bmo_kv_pages_plan(pages.handle, P(free), 3, P(lens), P(lens), P(table), 4, None, -1, None, None, None, None,
                               None) == 2
    assert L.bmo_kv_pages_plan(pages.handle, None, 3, P(lens), P(lens), P(table), 4, None, 0, None, None, None, None,
                               None) == 1
    assert "null" in pages.last_error()
    pages.close()

"""Plans that ask for no token's place: what is granted costs its pages, what is
refused nothing."""
import numpy as np
import pytest

from _pages import i32
from bmo_jetson_amd import KVPages
from test_gpu_pages_plan import Model, _compare, _device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,page,n_pages,width,most", [
    (1, 32, 4, 4, 40), (64, 32, 100, 9, 40), (300, 64, 900, 5, 90), (1024, 128, 900, 3, 100), (1500, 32, 2500, 6, 60),
    (2500, 64, 40000, 40, 1500)])
@pytest.mark.parametrize("said", [False, True])  # with what a caller's arrays would hold, or without a limit
def test_plans_without_places(gpu, n, page, n_pages, width, most, said):
    """Eight steps of growth, trims and ends against the model, with requests
    out of range among them and pools that run out."""
    from bmo_jetson_amd import lib
    pages = KVPages(1, n_pages, page, 1, 64)
    m = Model(n_pages, page, n, width)
    free, lens, table = _device(gpu, pages, n, width)
    start, status = (i32(gpu, np.zeros(size)) for size in (n + 1, n))
    r = np.random.default_rng(n)
    for step in range(8):
        kind = r.integers(0, 10, n)
        n_new = np.where(kind < 5, r.integers(0, most, n), np.where(kind < 7, 1, -r.integers(0, most, n)))
        if step == 3:
            n_new = np.where(kind < 8, -2**31 + 1, n_new)
        if step in (2, 5):
            n_new = np.where(kind == 0, 2**31 - 1, n_new)
        cap = int(np.maximum(n_new, 0).sum()) // 2 if said else 2**31 - 1
        cap = min(cap, 2**31 - 1)
        a = i32(gpu, n_new)
        P = lambda t: t.data_ptr()
        assert lib().bmo_kv_pages_plan(pages.handle, P(free), n, P(a), P(lens), P(table), width, P(start), cap, None, None,
                                       None, P(status), gpu.cuda.current_stream().cuda_stream) == 0
        want = _model_step(m, n_new, cap)
        assert start.cpu().tolist() == want[0] and status.cpu().tolist() == want[1]
        _compare(m, free, lens, table)
    pages.close()


def _model_step(m, n_new, cap):
    """Model.plan without the tokens of entries that it refuses (it lists every
    one), and with the starts' limit."""
    n_new = [int(x) for x in n_new]
    start, full, state = 0, [], []
    for b, x in enumerate(n_new):
        start += max(x, 0)
        full.append(x > 0 and start > cap)
        new = max(0, m.lens[b] + x)
        state.append(full[-1] or new > m.width * m.page)
    asked = [0 if s else x for x, s in zip(n_new, state)]
    _, status, _ = m.plan(asked, 2**62)
    starts = np.concatenate(([0], np.cumsum([max(x, 0) for x in n_new])))
    return [min(int(x), 2**31 - 1) for x in starts], [2 if s else x for s, x in zip(state, status)]


def test_a_request_out_of_range_costs_nothing(gpu):
    """2^31 - 1 tokens asked for and refused: once the time that an entry's
    tokens take (0.5 s), now that of its pages, none."""
    pages = KVPages(1, 64, 32, 1, 64)
    free, lens, table = _device(gpu, pages, 3, 8)
    status, stream = i32(gpu, np.zeros(3)), gpu.cuda.current_stream()
    took = []
    for n_new in ([1, 1, 1], [1, 2**31 - 1, 1]):
        a, b = gpu.cuda.Event(enable_timing=True), gpu.cuda.Event(enable_timing=True)
        n_new = i32(gpu, n_new)
        gpu.cuda.synchronize()
        a.record()
        pages.plan(free, n_new, lens, table, status=status, stream=stream)
        b.record()
        gpu.cuda.synchronize()
        took.append(a.elapsed_time(b))
    assert status.tolist() == [0, 2, 2] and lens.tolist() == [2, 1, 1]
    assert took[1] < 50, took  # ms
    pages.close()

"""Attention of one token per entry over its pages, plain and with the append,
against 64 bits (bounds in _pages.py)."""
import numpy as np
import pytest

from _pages import attention, check, i32, kv_rows, pool, rel, slot_of, to_type
from bmo_jetson_amd import KVPages, RingError

pytestmark = pytest.mark.gpu


def _work(gpu, pages, heads):
    return gpu.full((pages.workspace_bytes(heads) // 4,), float("nan"), device="cuda")


def _run(gpu, lens, page, heads, kv, dim, type_, window=0, seed=0, append=False, split=True, max_len=0, scale=0.0,
         table_edit=None, cache_edit=None):
    pages, cache, table = pool(gpu, lens, page, kv, dim, seed + 10)
    if cache_edit:
        cache_edit(pages, cache, table)
    if table_edit is not None:
        table = table_edit(table)
    n = len(lens)
    packed, x = to_type(gpu, np.concatenate([np.random.default_rng(seed).standard_normal((n, heads, dim)),
                                             kv_rows(seed + 1, n, 2 * kv, dim)], axis=1), type_)
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]
    out = gpu.zeros(n, heads, dim, dtype=q.dtype, device="cuda")
    args = dict(window=window, max_len=max_len, scale=scale, workspace=_work(gpu, pages, heads) if split else None,
                stream=gpu.cuda.current_stream())
    # and with a table of so many empty columns that the call is shaped for long entries
    long_table = np.concatenate([table, np.full((n, 2100 // page), -1)], axis=1)
    tables = [table] if table_edit is not None else [table, long_table]
    lens_d, outs = i32(gpu, lens), []
    if append:
        for t in tables:
            outs.append(gpu.full_like(out, float("nan")))
            pages.append_decode(0, lens_d, i32(gpu, t), q, k, v, outs[-1], **args)
        at = [slot_of(table, b, L - 1, page) if 0 < L else -1 for b, L in enumerate(lens)]
        cache.put(at, x[:, heads:heads + kv], x[:, heads + kv:])
        new = [gpu.zeros(n, kv, dim, device="cuda") for _ in range(2)]
        pages.gather(0, i32(gpu, at), *new, stream=gpu.cuda.current_stream())
        for got, want in zip(new, (cache.k, cache.v)):
            real = np.array(at) >= 0
            assert np.array_equal(got.cpu().numpy()[real], want[np.array(at)[real]])
    else:
        for t in tables:
            outs.append(gpu.full_like(out, float("nan")))
            pages.decode(0, lens_d, i32(gpu, t), q, outs[-1], **args)
    got = outs[0].double().cpu().numpy()
    refs, bounds = [], []
    for b, L in enumerate(lens):
        o, e = attention(cache, table[b], page, L, x[b:b + 1, :heads], [min(L, table.shape[1] * page) - 1], window, "decode",
                         type_, scale or None)
        refs.append(o[0])
        bounds.append(e[0])
    refs, bounds = np.stack(refs), np.stack(bounds)
    for x in outs:
        check(x.double().cpu().numpy(), refs, bounds, f"{lens} heads {heads}/{kv}x{dim} page {page} window {window}")
    pages.close()
    return got, refs


@pytest.mark.parametrize("dim,page", [(128, 16), (128, 64), (64, 32), (64, 256)])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (8, 2), (12, 2), (10, 2), (16, 1), (40, 2)])
@pytest.mark.parametrize("append", [False, True])
def test_lengths_and_head_layouts(gpu, dim, page, heads, kv, append):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 63, 65, 200]
    got, refs = _run(gpu, lens, page, heads, kv, dim, "float32", append=append, split=False)
    assert not got[0].any()
    # far within the bound on the whole: fp32 arithmetic, not 16 bits
    assert rel(got, refs) < 5e-6


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (16, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("append", [False, True])
def test_types_and_split_entries(gpu, type_, heads, kv, dim, append):
    # one long entry among short ones: its steps are cut in many runs
    lens = [5000, 0, 40, 1, 999, 257]
    _run(gpu, lens, 64, heads, kv, dim, type_, append=append)
    _run(gpu, lens, 64, heads, kv, dim, type_, append=append, split=False)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 640])
@pytest.mark.parametrize("append", [False, True])
def test_windows(gpu, window, append):
    _run(gpu, [1, 2, 32, 99, 100, 101, 640, 641, 700, 1300], 32, 4, 2, 64, "float32", window=window, append=append)


@pytest.mark.parametrize("n,heads,kv", [(1, 1, 1), (65, 2, 2), (200, 4, 1), (257, 1, 1)])
def test_many_and_few_entries(gpu, n, heads, kv):
    r = np.random.default_rng(n)
    lens = [9000 if n == 1 else int(x) for x in r.integers(0, 600, n)]
    _run(gpu, lens, 32, heads, kv, 64, "float32", max_len=max(lens))


def test_max_len_is_a_hint_and_scale_is_used(gpu):
    _run(gpu, [700, 3, 1200], 64, 4, 4, 128, "float32", max_len=10)  # longer than said
    _run(gpu, [700, 3, 1200], 64, 4, 4, 128, "float32", max_len=1 << 30)
    _run(gpu, [300, 3], 64, 4, 4, 128, "float32", scale=0.02)


def test_large_scores_and_small_scales(gpu):
    """Keys and values of very different sizes, block by block."""
    def edit(pages, cache, table):
        n = len(cache.k)
        k, v = kv_rows(91, n, 2, 128), kv_rows(92, n, 2, 128)
        v[:, :, :32] *= 1e-4
        v[:, :, 32:64] *= 1e4
        k[:, :, 96:] *= 30.0
        cache.put(np.arange(n), k, v)
        pages.append(0, i32(gpu, np.arange(n)), gpu.from_numpy(k).cuda(), gpu.from_numpy(v).cuda(),
                     stream=gpu.cuda.current_stream())
    for heads in (2, 16):
        _run(gpu, [600, 33], 64, heads, 2, 128, "float32", cache_edit=edit)


def _spoil(gpu, pages, cache, slots, kv, dim):
    """Infinite and NaN blocks in slots (their positions are to be masked)."""
    x = np.full((len(slots), kv, dim), np.nan, dtype=np.float32)
    x[::2] = np.inf
    pages.append(0, i32(gpu, slots), gpu.from_numpy(x).cuda(), gpu.from_numpy(x).cuda(),
                 stream=gpu.cuda.current_stream())


@pytest.mark.parametrize("heads", [2, 4, 32])
@pytest.mark.parametrize("window", [0, 50])
def test_what_masked_positions_hold_does_not_show(gpu, heads, window):
    lens, page, kv, dim = [70, 1, 300], 64, 2, 128

    def edit(pages, cache, table):
        used = set()
        for b, L in enumerate(lens):
            lo = max(0, L - window) if window else 0
            used |= {slot_of(table, b, p, page) for p in range(lo, L)}
        _spoil(gpu, pages, cache, np.array(sorted(set(range(len(cache.k))) - used)), kv, dim)
    for append in (False, True):
        _run(gpu, lens, page, heads, kv, dim, "float32", window=window, cache_edit=edit, append=append)


def test_bad_page_ids_are_masked(gpu):
    def edit(table):
        t = table.copy()
        t[0, 1] = -1
        t[1, 0] = 2**31 - 1
        t[2, :] = -2**31
        t[3, 2] = 10**6
        return t
    for heads in (2, 16):
        got, _ = _run(gpu, [200, 40, 90, 180], 64, heads, 2, 128, "float32", table_edit=edit)
        assert not got[1].any() and not got[2].any()


def test_append_to_a_bad_page_is_dropped(gpu):
    pages, cache, table = pool(gpu, [40, 64], 32, 2, 64, 3)
    before = [gpu.zeros(len(cache.k), 2, 64, device="cuda") for _ in range(2)]
    every = i32(gpu, np.arange(len(cache.k)))
    pages.gather(0, every, *before)
    t = table.copy()
    t[0, 1], t[1, 1] = -1, pages.n_pages
    q = gpu.randn(2, 4, 64, device="cuda")
    out = gpu.zeros_like(q)
    pages.append_decode(0, i32(gpu, [40, 64]), i32(gpu, t), q, q[:, :2], q[:, 2:], out)
    after = [gpu.zeros_like(x) for x in before]
    pages.gather(0, every, *after)
    assert all(gpu.equal(a, b) for a, b in zip(before, after)) and bool(out.isfinite().all())
    pages.close()


def test_nan_in_one_query_stays_in_its_rows(gpu):
    pages, cache, table = pool(gpu, [100, 50], 64, 2, 128, 5)
    for heads in (4, 16):
        q = gpu.randn(2, heads, 128, device="cuda")
        out, want = gpu.zeros_like(q), gpu.zeros_like(q)
        pages.decode(0, i32(gpu, [100, 50]), i32(gpu, table), q, want)
        q[0, 1, 77] = float("nan")
        q[1, heads - 1, 0] = float("inf")
        pages.decode(0, i32(gpu, [100, 50]), i32(gpu, table), q, out)
        bad = gpu.zeros(2, heads, dtype=gpu.bool, device="cuda")
        bad[0, 1] = bad[1, heads - 1] = True
        assert bool(out[bad].isnan().all()) and gpu.equal(out[~bad], want[~bad])
    pages.close()


def test_lengths_past_the_table(gpu):
    _run(gpu, [100, 64, 30], 64, 2, 2, 64, "float32", table_edit=lambda t: t[:, :1].copy())


def test_other_layers_and_streams(gpu):
    pages, cache, table = pool(gpu, [90, 10], 32, 2, 64, 7, layers=3, layer=2)
    lens, t = i32(gpu, [90, 10]), i32(gpu, table)
    q, x = to_type(gpu, np.random.default_rng(1).standard_normal((2, 6, 64)), "float32")
    out = gpu.zeros_like(q)
    gpu.cuda.synchronize()
    s = gpu.cuda.Stream()
    with gpu.cuda.stream(s):
        pages.decode(2, lens, t, q, out, stream=s)
    s.synchronize()
    for b, L in enumerate((90, 10)):
        o, e = attention(cache, table[b], 32, L, x[b:b + 1], [L - 1], 0, "decode", "float32")
        check(out[b:b + 1].cpu().numpy(), o, e)
    pages.decode(0, lens, t, q, out)  # a layer of zeros
    gpu.cuda.synchronize()
    assert not out.any()
    pages.close()


def test_two_graphs_with_their_own_workspaces(gpu):
    """Captured and replayed in turn, between eager calls; the same bits every time."""
    calls = []
    for heads, seed in ((4, 20), (16, 30)):
        pages, cache, table = pool(gpu, [3000, 100, 1700], 64, 2, 128, seed)
        q = gpu.randn(3, heads, 128, device="cuda")
        lens, t = i32(gpu, [3000, 100, 1700]), i32(gpu, table)
        out, work = gpu.zeros_like(q), _work(gpu, pages, heads)
        call = lambda o, w, p=pages, a=lens, b=t, q=q: p.decode(0, a, b, q, o, workspace=w,
                                                               stream=gpu.cuda.current_stream())
        graph, side = gpu.cuda.CUDAGraph(), gpu.cuda.Stream()
        side.wait_stream(gpu.cuda.current_stream())
        with gpu.cuda.stream(side), gpu.cuda.graph(graph, stream=side):
            call(out, work)
        gpu.cuda.current_stream().wait_stream(side)
        eager = gpu.zeros_like(q)
        call(eager, _work(gpu, pages, heads))
        calls.append((graph, out, eager, q, call, pages, work))  # (a graph keeps no tensor alive)
    for step in range(5):
        for graph, out, eager, q, call, pages, _ in calls:
            q.mul_(1.1)
            call(eager, None if step == 3 else _work(gpu, pages, q.shape[1]))
            graph.replay()
            gpu.cuda.synchronize()
            if step == 3:
                assert gpu.allclose(out, eager, rtol=1e-4, atol=1e-5)
            else:
                assert gpu.equal(out, eager)
    for c in calls:
        c[5].close()


def test_refusals(gpu):
    pages = KVPages(1, 4, 32, 2, 64)
    lens, table = i32(gpu, [3, 4]), i32(gpu, [[0, 1], [2, 3]])
    q = gpu.zeros(2, 4, 64, device="cuda")
    out = gpu.zeros_like(q)
    with pytest.raises(RingError, match="layer"):
        pages.decode(1, lens, table, q, out)
    with pytest.raises(RingError, match="multiple"):
        pages.decode(0, lens, table, q[:, :3].contiguous(), out[:, :3].contiguous())
    for kw in ({"window": -1}, {"max_len": -1}, {"scale": float("inf")}):
        with pytest.raises(RingError):
            pages.decode(0, lens, table, q, out, **kw)
    with pytest.raises(ValueError):
        pages.decode(0, lens, table, q[:1], out)
    with pytest.raises(ValueError):
        pages.decode(0, lens, table, q, out.half())
    with pytest.raises(ValueError):
        pages.append_decode(0, lens, table, q, q[:, :2].half(), q[:, 2:].half(), out)
    with pytest.raises(RingError, match="aligned"):
        pages.decode(0, lens, table, gpu.zeros(2 * 4 * 64 + 1, device="cuda")[1:].view(2, 4, 64), out)
    assert pages.workspace_bytes(3) == 0 and pages.workspace_bytes(4) > 0
    pages.close()

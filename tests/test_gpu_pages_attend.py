"""Ragged rows over their entries' pages, causal chunks and cross attention,
against 64 bits (bounds in _pages.py)."""
import numpy as np
import pytest

from _pages import attention, check, i32, kv_rows, pool, rel, slot_of, to_type
from bmo_jetson_amd import KVPages, RingError

pytestmark = pytest.mark.gpu


MORE = 256  # rows behind the last, so that a call can be said to have so many an entry


def _tiles(gpu, start, lens, table, rows, group, kv):
    """The same call with as many empty entries and as large a hint as make it
    one of tiles (few rows are taken in sets of columns): q_start, lens, table,
    max_rows.  q has MORE rows behind the last."""
    more, most = 64 - len(lens), max(MORE, *rows)
    units = 64 * kv
    assert more >= 0 and -(-most * group // 16) * units >= max(1024, 2 * -(-most * group // 128) * units + 1)
    start = np.concatenate((start, [start[-1]] * more))
    return (i32(gpu, start), i32(gpu, np.concatenate((lens, [0] * more))),
            i32(gpu, np.concatenate((table, np.full((more, table.shape[1]), -1)))), most)


def _calls(gpu, start, lens, table, rows, tiles, group=1, kv=1):
    if tiles:
        return _tiles(gpu, start, lens, table, rows, group, kv)
    return i32(gpu, start), i32(gpu, lens), i32(gpu, table), max(rows)


def _run(gpu, rows, lens, page, heads, kv, dim, type_="bfloat16", causal=True, window=0, seed=0, max_rows=None, tail=3,
         table_edit=None, cache_edit=None, workspace=True, scale=0.0, gap=1, tol=True):
    pages, cache, table = pool(gpu, lens, page, kv, dim, seed + 40)
    if cache_edit:
        cache_edit(pages, cache, table)
    if table_edit is not None:
        table = table_edit(table)
    total = sum(rows)
    packed, x = to_type(gpu, np.random.default_rng(seed).standard_normal((total + tail + MORE, heads + gap, dim)), type_)
    start = np.concatenate(([0], np.cumsum(rows)))
    work = None
    if workspace:
        work = gpu.full((pages.workspace_bytes(heads) // 4,), float("nan"), device="cuda")
    calls = [_calls(gpu, start, lens, table, [max(rows) if max_rows is None else max_rows], False)]
    # with a table of so many empty columns that sets of columns are shaped for long entries
    calls.append(_calls(gpu, start, lens, np.concatenate([table, np.full((len(lens), 2100 // page), -1)], axis=1),
                        [calls[0][3]], False))
    if table_edit is not None:
        calls.pop()  # (an edited table's own width counts)
    if len(lens) <= 64:
        calls.append(_tiles(gpu, start, lens, table, rows, heads // kv, kv))
    results = []
    for start_d, lens_d, table_d, most in calls:
        q = packed[:, :heads] if len(lens_d) > len(lens) else packed[:total + tail, :heads]
        out = gpu.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
        pages.attend(0, start_d, lens_d, table_d, q, out, causal=causal, window=window, scale=scale, max_rows=most,
                     workspace=work, stream=gpu.cuda.current_stream())
        results.append(out.double().cpu().numpy())
        assert (results[-1][total:] == 7.0).all()  # rows behind the last
    refs, bounds = np.zeros((total, heads, dim)), np.zeros((total, heads, dim))
    for b, (n, L) in enumerate(zip(rows, lens)):
        L = min(L, table.shape[1] * page)
        last = [L - n + i if causal else L - 1 for i in range(n)]
        a, e = attention(cache, table[b], page, L, x[start[b]:start[b + 1], :heads], last, window, "attend", type_,
                         scale or None)
        refs[start[b]:start[b + 1]], bounds[start[b]:start[b + 1]] = a, e
    for got in results:
        if tol:
            check(got[:total], refs, bounds, f"rows {rows} lens {lens} heads {heads}/{kv}x{dim} page {page} causal {causal}")
            # on the whole: the output's rounding, and 16-bit operands
            assert rel(got[:total], refs) < {"bfloat16": 2.0**-8, "float16": 2.0**-9}[type_]
    pages.close()
    return got[:total], refs


@pytest.mark.parametrize("dim,page", [(128, 16), (128, 128), (64, 32), (64, 64)])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 2), (6, 2), (16, 1), (5, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_lengths_and_head_layouts(gpu, dim, page, heads, kv, causal):
    _run(gpu, [1, 0, 5, 33, 130, 17, 64], [1, 50, 70, 33, 200, 16, 257], page, heads, kv, dim, causal=causal)


@pytest.mark.parametrize("type_", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [[1], [2, 8], [31, 32, 33], [127, 128, 129], [300]])
@pytest.mark.parametrize("causal", [True, False])
def test_types_and_tiles(gpu, type_, rows, causal):
    _run(gpu, rows, [n + 90 * i for i, n in enumerate(rows)], 64, 4, 2, 128, type_, causal=causal)


@pytest.mark.parametrize("window", [1, 30, 64, 65, 200])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(gpu, window, causal):
    _run(gpu, [100, 3, 150], [100, 300, 400], 32, 4, 2, 64, window=window, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing(gpu, causal):
    # more rows than positions, and no positions at all
    got, _ = _run(gpu, [40, 9, 4], [10, 0, 50], 32, 2, 2, 64, causal=causal)
    assert not got[40:49].any()
    if causal:
        assert not got[:30].any() and got[30:40].any()


def test_few_rows_of_long_entries(gpu):
    for causal in (True, False):
        for heads, kv in ((2, 2), (8, 1), (16, 1)):
            _run(gpu, [1, 3, 2], [4000, 20, 2500], 64, heads, kv, 128, causal=causal, type_="float16")
            _run(gpu, [1, 3, 2], [4000, 20, 2500], 64, heads, kv, 128, causal=causal, workspace=False)


def test_many_entries(gpu):
    r = np.random.default_rng(3)
    rows = [int(x) for x in r.integers(0, 40, 150)]
    _run(gpu, rows, [n + int(x) for n, x in zip(rows, r.integers(0, 60, 150))], 32, 2, 1, 64, max_rows=0)
    _run(gpu, rows, [n + int(x) for n, x in zip(rows, r.integers(0, 60, 150))], 32, 2, 1, 64)


def test_scale(gpu):
    _run(gpu, [20], [90], 64, 2, 2, 64, scale=0.05)


def _spoil(gpu, pages, slots, kv, dim):
    x = np.full((len(slots), kv, dim), np.nan, dtype=np.float32)
    x[::2] = np.inf
    pages.append(0, i32(gpu, slots), gpu.from_numpy(x).cuda(), gpu.from_numpy(x).cuda(),
                 stream=gpu.cuda.current_stream())


@pytest.mark.parametrize("rows", [[2, 1], [60, 200]])
@pytest.mark.parametrize("window", [0, 70])
def test_what_masked_positions_hold_does_not_show(gpu, rows, window):
    lens, page, kv, dim = [rows[0] + 100, rows[1]], 64, 2, 128

    def edit(pages, cache, table):
        used = set()
        for b, (n, L) in enumerate(zip(rows, lens)):
            lo = max(0, L - n + 1 - window) if window else 0
            used |= {slot_of(table, b, p, page) for p in range(lo, L)}
        _spoil(gpu, pages, np.array(sorted(set(range(len(cache.k))) - used)), kv, dim)
    _run(gpu, rows, lens, page, 4, kv, dim, window=window, cache_edit=edit)


@pytest.mark.parametrize("rows,at", [(150, 90), (3, 98)])
@pytest.mark.parametrize("tiles", [False, True])
def test_a_value_that_is_not_finite_reaches_only_rows_that_see_it(gpu, rows, at, tiles):
    """V block 1 of position `at` is infinite: rows before it are as they are
    without it, later ones are not finite in that block alone."""
    page, kv, dim, heads = 32, 1, 128, 2
    L = max(rows, 100)
    pages, cache, table = pool(gpu, [L], page, kv, dim, 60)
    q = gpu.randn(rows + MORE * tiles, heads, dim, device="cuda").bfloat16()
    start, lens, t, most = _calls(gpu, [0, rows], [L], table, [rows], tiles, 2)
    want, out = gpu.zeros_like(q), gpu.zeros_like(q)
    pages.attend(0, start, lens, t, q, want, max_rows=most)
    slot = i32(gpu, [slot_of(table, 0, at, page)])
    k, v = (gpu.zeros(1, kv, dim // 32, 18, dtype=gpu.uint8, device="cuda") for _ in range(2))
    pages.gather(0, slot, k, v)
    v[0, 0, 1, :2] = gpu.tensor([0, 0x7C], dtype=gpu.uint8)
    pages.append(0, slot, k, v)
    pages.attend(0, start, lens, t, q, out, max_rows=most)
    gpu.cuda.synchronize()
    out, want = out[:rows], want[:rows]
    sees = L - rows + np.arange(rows) >= at
    assert 0 < sees.sum() < rows
    sees = gpu.from_numpy(sees).cuda()
    assert gpu.equal(out[~sees], want[~sees])
    assert not bool(out[sees][:, :, 32:64].isfinite().any())
    rest = [c for c in range(dim) if not 32 <= c < 64]
    assert gpu.equal(out[sees][:, :, rest], want[sees][:, :, rest])
    pages.close()


@pytest.mark.parametrize("rows", [[2, 1, 2], [70, 33, 40]])
def test_bad_page_ids_are_masked(gpu, rows):
    def edit(table):
        t = table.copy()
        t[0, 1], t[1, 0], t[2, :] = -1, 10**8, -2**31
        return t
    got, _ = _run(gpu, rows, [200, 60, 90], 64, 4, 2, 128, table_edit=edit, causal=False)
    assert not got[rows[0]:].any()


@pytest.mark.parametrize("tiles", [False, True])
def test_nan_in_one_query_stays_in_its_row(gpu, tiles):
    pages, cache, table = pool(gpu, [100], 64, 2, 128, 5)
    q = gpu.randn(50 + MORE * tiles, 4, 128, device="cuda").half()
    out, want = gpu.zeros_like(q), gpu.zeros_like(q)
    *args, most = _calls(gpu, [0, 50], [100], table, [50], tiles, 2, 2)
    pages.attend(0, *args, q, want, max_rows=most)
    q[7, 2, 3] = float("nan")
    pages.attend(0, *args, q, out, max_rows=most)
    bad = gpu.zeros(q.shape[:2], dtype=gpu.bool, device="cuda")
    bad[7, 2] = True
    assert bool(out[bad].isnan().all()) and gpu.equal(out[~bad], want[~bad])
    pages.close()


@pytest.mark.parametrize("tiles", [False, True])
def test_starts_that_are_no_running_sum(gpu, tiles):
    """Entries whose rows are not within q are skipped."""
    pages, cache, table = pool(gpu, [50, 50, 50], 64, 2, 64, 8)
    n = 20 + MORE * tiles
    q = gpu.randn(n, 2, 64, device="cuda").half()
    for start in ([0, n + 10, 5, 10], [-4, 5, 10, 20], [2**31 - 1, 0, 2**31 - 1, -2**31]):
        out = gpu.full_like(q, 7.0)
        *args, most = _calls(gpu, start, [50] * 3, table, [20], tiles, 1, 2)
        pages.attend(0, *args, q, out, causal=False, max_rows=most)
        gpu.cuda.synchronize()
        if start[0] == 0:
            assert bool((out[:5] == 7.0).all()) and bool((out[10:] == 7.0).all())
    pages.close()


@pytest.mark.parametrize("tiles", [False, True])
def test_replayed_from_a_graph(gpu, tiles):
    for rows, heads in (([40, 200], 4), ([1, 2], 4)):
        lens = [900, 250]
        pages, cache, table = pool(gpu, lens, 64, 2, 128, 9)
        q = gpu.randn(sum(rows) + MORE * tiles, heads, 128, device="cuda").half()
        start, ln, t, most = _calls(gpu, [0, rows[0], sum(rows)], lens, table, rows, tiles, 2, 2)
        work, work2 = (gpu.zeros(pages.workspace_bytes(heads), dtype=gpu.uint8, device="cuda") for _ in range(2))
        out, eager = gpu.zeros_like(q), gpu.zeros_like(q)
        graph, side = gpu.cuda.CUDAGraph(), gpu.cuda.Stream()
        side.wait_stream(gpu.cuda.current_stream())
        with gpu.cuda.stream(side), gpu.cuda.graph(graph, stream=side):
            pages.attend(0, start, ln, t, q, out, max_rows=most, workspace=work, stream=gpu.cuda.current_stream())
        gpu.cuda.current_stream().wait_stream(side)
        for _ in range(4):
            q.mul_(1.05)
            graph.replay()
            pages.attend(0, start, ln, t, q, eager, max_rows=most, workspace=work2, stream=gpu.cuda.current_stream())
            gpu.cuda.synchronize()
            assert gpu.equal(out, eager) and bool(out.any())
        pages.close()


def test_refusals(gpu):
    pages = KVPages(1, 4, 32, 2, 64)
    lens, table, start = i32(gpu, [3, 4]), i32(gpu, [[0, 1], [2, 3]]), i32(gpu, [0, 1, 2])
    q = gpu.zeros(2, 4, 64, device="cuda").half()
    with pytest.raises(RingError, match="fp16 or bf16"):
        pages.attend(0, start, lens, table, q.float(), q.float())
    with pytest.raises(RingError, match="layer"):
        pages.attend(-1, start, lens, table, q, q.clone())
    for kw in ({"window": -1}, {"max_len": -1}, {"max_rows": -1}, {"scale": float("nan")}):
        if "scale" in kw:
            pages.attend(0, start, lens, table, q, q.clone(), **kw)  # not positive: the default
            continue
        with pytest.raises(RingError):
            pages.attend(0, start, lens, table, q, q.clone(), **kw)
    with pytest.raises(ValueError):
        pages.attend(0, start[:2], lens, table, q, q.clone())
    pages.attend(0, start, lens, table, q[:0], q[:0].clone())  # nothing to do
    gpu.cuda.synchronize()
    pages.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (16, 1)])
@pytest.mark.parametrize("window", [0, 45])
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows_in_sets_of_columns(gpu, dim, heads, kv, window, causal):
    """Entries whose rows share sets of 4, 8 or 16 columns, full and not, and
    ends and windows that differ from row to row."""
    for type_ in ("float16", "bfloat16"):
        _run(gpu, [7, 1, 0, 17, 4], [300, 1, 5, 17, 0], 64, heads, kv, dim, type_, causal=causal, window=window)


def test_few_and_many_rows_agree(gpu):
    """An entry's rows alone, by sets of columns, and among so many that the
    call is taken by tiles."""
    pages, cache, table = pool(gpu, [700] * 70, 64, 4, 128, 9)
    q = gpu.randn(70 * 48, 4, 128, device="cuda").half()
    lens, t = i32(gpu, [700] * 70), i32(gpu, table)
    a, b = gpu.zeros_like(q), gpu.zeros_like(q)
    stream = gpu.cuda.current_stream()
    pages.attend(0, i32(gpu, np.arange(71) * 48), lens, t, q, a, max_rows=48, stream=stream)
    for i in (0, 33, 69):
        rows = slice(48 * i, 48 * i + 48)
        pages.attend(0, i32(gpu, [0, 48]), lens[:1], t[i:i + 1], q[rows], b[rows], max_rows=48, stream=stream)
        # both are within a rounding (2^-11) and the operands' (2^-10) of the exact ones
        assert rel(b[rows].double().cpu().numpy(), a[rows].double().cpu().numpy()) < 2.0**-9
    pages.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tiles", [False, True])
def test_fp16_scores_are_as_exact_as_fp32(gpu, dim, tiles):
    """Queries 16 times as large: keys rounded to fp16 would be off by 2^-12 of
    scores around 16 to 100.  Three roundings to 11 bits remain (the output, V,
    the weights), each at most 2^-11 / sqrt(3) of the whole in the mean square
    when they are independent: 2^-11 together."""
    rows, lens = [40, 300], [700, 700]
    pages, cache, table = pool(gpu, lens, 64, 2, dim, 77)
    q, x = to_type(gpu, 16 * np.random.default_rng(6).standard_normal((340, 4, dim)), "float16")
    out = gpu.zeros_like(q)
    *args, most = _calls(gpu, [0, 40, 340], lens, table, rows, tiles, 2, 2)
    pages.attend(0, *args, q, out, max_rows=most, stream=gpu.cuda.current_stream())
    ref = np.concatenate([attention(cache, table[b], 64, 700, x[at:at + n], list(range(700 - n, 700)), 0, "attend",
                                    "float16")[0] for b, (at, n) in enumerate(((0, 40), (40, 300)))])
    assert rel(out.double().cpu().numpy(), ref) < 2.0**-11
    pages.close()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("long", [False, True])
def test_rows_that_see_nothing_are_zeros_whatever_their_queries_hold(gpu, tiles, long):
    """A causal chunk longer than its entry: NaN and infinities in the rows
    before position 0, beside rows that see something."""
    lens, rows = [3000 if long else 5, 5], [40, 40]
    pages, cache, table = pool(gpu, lens, 64, 2, 128, 31)
    q = gpu.randn(80 + MORE * tiles, 4, 128, device="cuda").half()
    want, out = gpu.zeros_like(q), gpu.full_like(q, 7.0)
    *args, most = _calls(gpu, [0, 40, 80], lens, table, rows, tiles, 2, 2)
    work = gpu.zeros(pages.workspace_bytes(4), dtype=gpu.uint8, device="cuda")
    pages.attend(0, *args, q, want, max_rows=most, workspace=work)
    blind = gpu.zeros(len(q), dtype=gpu.bool, device="cuda")
    blind[40:75] = True
    if not long:
        blind[:35] = True
    q[blind] = float("nan")
    q[42] = float("inf")
    pages.attend(0, *args, q, out, max_rows=most, workspace=work)
    gpu.cuda.synchronize()
    sees = ~blind
    sees[80:] = False
    assert not bool(out[blind].any()) and gpu.equal(out[sees], want[sees])
    pages.close()


def test_more_rows_than_said_leave_the_others_whole(gpu):
    for rows, said in (([300, 2, 2, 2], 2), ([2, 700, 300, 33], 40)):
        lens = [700] * 64
        pages, cache, table = pool(gpu, lens, 64, 8, 64, 12)
        rows = rows + [0] * 60
        start = np.concatenate(([0], np.cumsum(rows)))
        q = gpu.randn(sum(rows), 16, 64, device="cuda").half()
        want, out = gpu.zeros_like(q), gpu.full_like(q, 7.0)
        args = (0, i32(gpu, start), i32(gpu, lens), i32(gpu, table), q)
        pages.attend(*args, want, max_rows=max(rows), stream=gpu.cuda.current_stream())
        pages.attend(*args, out, max_rows=said, stream=gpu.cuda.current_stream())
        for b, n in enumerate(rows):
            part = slice(start[b], start[b] + min(n, said))
            # (the two calls may be shaped differently: roundings of 16-bit operands)
            assert rel(out[part].double().cpu().numpy(), want[part].double().cpu().numpy()) < 2.0**-9
        pages.close()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [65520.0, 7e4, 5e5, float("inf")])
def test_values_past_fp16_at_masked_positions_do_not_show(gpu, tiles, dim, value):
    """What an fp32 request may have left in a page: scales within fp16 whose
    values are not.  A row that sees one is not finite in that block."""
    page, kv, heads, rows = 64, 1, 2, 60
    pages, cache, table = pool(gpu, [200], page, kv, dim, 4)
    q = gpu.randn(rows + MORE * tiles, heads, dim, device="cuda").bfloat16()
    *args, most = _calls(gpu, [0, rows], [150], table, [rows], tiles, 2)
    want, out = gpu.zeros_like(q), gpu.zeros_like(q)
    pages.attend(0, *args, q, want, max_rows=most)
    far = np.array([slot_of(table, 0, p, page) for p in range(150, 200)])
    x = gpu.full((len(far), kv, dim), value, device="cuda")
    x[::2] *= -1
    pages.append(0, i32(gpu, far), x, x)
    pages.attend(0, *args, q, out, max_rows=most)
    assert bool(want.any()) and gpu.equal(out, want)
    # at position 120, in V's last block alone: rows 0..29 end before it
    k, v = gpu.zeros(1, kv, dim, device="cuda"), gpu.zeros(1, kv, dim, device="cuda")
    at = i32(gpu, [slot_of(table, 0, 120, page)])
    pages.append(0, at, k, v)
    pages.attend(0, *args, q, want, max_rows=most)
    v[0, 0, -3] = value
    pages.append(0, at, k, v)
    pages.attend(0, *args, q, out, max_rows=most)
    assert gpu.equal(out[:30], want[:30]) and gpu.equal(out[:, :, :-32], want[:, :, :-32])
    if tiles or not np.isfinite(value):
        assert not bool(out[30:rows, :, -32:].isfinite().all(-1).any())
    pages.close()

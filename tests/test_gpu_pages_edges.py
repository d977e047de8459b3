"""The paged cache at the edges of its tables, its scales and its queries."""
import numpy as np
import pytest

from _pages import HALF_STEP, attention, check, i32, kv_rows, pool, rel, slot_of, to_type

pytestmark = pytest.mark.gpu

# A result as a whole, in the mean square.  A rounding is at most half a step,
# relative to the value, and 1 / sqrt(3) of that in the mean square.  fp16 rows:
# the output's rounding and the weight's, 2^-11 sqrt(2 / 3); bf16 rows: 2^-8 /
# sqrt(3) and the weight's 2^-11.  fp32: sums of some hundred roundings of 2^-24.
WHOLE = {"float32": 5e-6, "float16": 2.0**-11, "bfloat16": 2.0**-8}
# An output below the type's normal range ends at a fixed step, half of which is
# what rounding can cost there whatever the value: fp16's step is 2^-24.
LEAST = {"float32": 0.0, "float16": 2.0**-25, "bfloat16": 0.0}


def check_whole(got, ref, type_):
    off = np.linalg.norm(got - ref)
    assert off < WHOLE[type_] * np.linalg.norm(ref) + LEAST[type_] * ref.size**0.5, rel(got, ref)


def decode_reference(cache, table_row, page, length, q, type_, scale=None):
    """(out, bound) of rows q that see all of an entry's positions, in 64 bits.
    A query is within 2^-22 of each of its own elements (fp32: two fp16 parts,
    each rounded, 2^-11 of 2^-11; 16-bit rows are exact) and within 2^-39 of its
    largest (the parts end at 2^-24, half a step of that is 2^-25, the largest
    is scaled past 2^14); a score sums 32 products in a block and up to 4 blocks
    in fp32, 40 roundings of 2^-24, scaled, shifted by the maximum and raised
    (4 more).  So it is off by e = (2^-22 + 44 2^-24) sum|q k| + 2^-39 max|q|
    sum|k|, which moves a weight by e of itself and the sum by as much.  The
    weighted sum itself: two parts of a weight (2^-22) and sums in fp32, within
    2^-16 of 16 sum p|d| as in _pages; of 16-bit rows one part, 2^-11."""
    n, heads, dim = q.shape
    group = heads // cache.k.shape[1]
    scale = dim**-0.5 if scale is None else scale
    at = np.array([slot_of([table_row], 0, p, page) for p in range(length)])
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        for h in range(heads):
            k, v, d = cache.k[at, h // group], cache.v[at, h // group], np.abs(cache.d[at, h // group])
            s = k @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            off = (2.0**-22 + 44 * 2.0**-24) * (np.abs(k) @ np.abs(q[i, h])).max() * scale
            off += 2.0**-39 * np.abs(q[i, h]).max() * np.abs(k).sum(axis=1).max() * scale
            b = (2 * off + (0 if type_ == "float32" else 2.0**-11)) * (p @ np.abs(v))
            b += 2.0**-16 * 16 * np.repeat(p @ d, 32)
            out[i, h] = p @ v
            bound[i, h] = b + HALF_STEP[type_] * (np.abs(out[i, h]) + b) + LEAST[type_]
    return out, bound


def refill(gpu, pages, cache, k, v):
    """Every slot of layer 0 anew."""
    every = np.arange(len(cache.k))
    cache.put(every, k, v)
    pages.append(0, i32(gpu, every), *(gpu.from_numpy(x).cuda() for x in (k, v)), stream=gpu.cuda.current_stream())


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 2, 128), (16, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("past", [1, 30, 2**31 - 1])
def test_a_token_past_the_table_is_dropped(gpu, heads, kv, dim, past):
    """An entry longer than its table's room (by `past`, or as long as an int
    goes) beside one that fills the table and one within it."""
    page = 32
    pages, cache, table = pool(gpu, [64, 64, 40], page, kv, dim, 3)
    long = [min(64 + past, 2**31 - 1), 64, 40]
    every = np.arange(len(cache.k))
    packed, x = to_type(gpu, np.concatenate([np.random.default_rng(1).standard_normal((3, heads, dim)),
                                             kv_rows(2, 3, 2 * kv, dim)], axis=1), "float32")
    q, k, v = packed.split([heads, kv, kv], dim=1)
    out, plain = gpu.zeros(3, heads, dim, device="cuda"), gpu.zeros(3, heads, dim, device="cuda")
    stream = gpu.cuda.current_stream()
    pages.append_decode(0, i32(gpu, long), i32(gpu, table), q, k, v, out, stream=stream)
    cache.put([int(table[1, 1]) * page + 31, int(table[2, 1]) * page + 7], x[1:, heads:heads + kv], x[1:, heads + kv:])
    got = [gpu.zeros(len(every), kv, dim, device="cuda") for _ in range(2)]
    pages.gather(0, i32(gpu, every), *got, stream=stream)
    for g, want in zip(got, (cache.k, cache.v)):
        assert np.array_equal(g.cpu().numpy(), want)
    for b, n in enumerate((64, 64, 40)):  # attended as far as the table goes
        ref, bound = attention(cache, table[b], page, n, x[b:b + 1, :heads], [n - 1], 0, "decode", "float32")
        check(out[b:b + 1].cpu().numpy(), ref, bound, f"entry {b}")
    pages.decode(0, i32(gpu, long), i32(gpu, table), q, plain, stream=stream)
    assert gpu.equal(out, plain)
    pages.close()


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (3, 1, 64), (16, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("big", [30, 300, 3000])
def test_a_query_channel_far_above_the_rest(gpu, type_, heads, kv, dim, big):
    """One channel of the query `big` times the others, against keys that hold
    nothing there: the other channels keep their own precision, in decode, in
    few rows and in tiles."""
    page, length = 64, 600
    pages, cache, table = pool(gpu, [length], page, kv, dim, 5)
    k, v = kv_rows(3, len(cache.k), kv, dim), kv_rows(4, len(cache.k), kv, dim)
    k[:, :, 41] = 0.0
    refill(gpu, pages, cache, k, v)
    x = np.random.default_rng(1).standard_normal((1, heads, dim))
    x[:, :, 41] = big
    q, x = to_type(gpu, x, type_)
    lens, t, stream = i32(gpu, [length]), i32(gpu, table), gpu.cuda.current_stream()
    ref, bound = decode_reference(cache, table[0], page, length, x, type_)
    out = gpu.zeros_like(q)
    pages.decode(0, lens, t, q, out, stream=stream)
    got = out.double().cpu().numpy()
    check(got, ref, bound, "decode")
    check_whole(got, ref, type_)
    if type_ != "float32":
        out.zero_()
        pages.attend(0, i32(gpu, [0, 1]), lens, t, q, out, max_rows=1, stream=stream)
        got = out.double().cpu().numpy()
        check(got, ref, bound, "few rows")
        check_whole(got, ref, type_)
        # and as one of so many entries and rows that they are taken in tiles
        q = gpu.cat([q, q.new_zeros(2000, heads, dim)])
        out, n = gpu.zeros_like(q), 64
        pages.attend(0, i32(gpu, [0] + [1] * n), i32(gpu, [length] + [0] * (n - 1)),
                     gpu.cat([t, t.new_full((n - 1, t.shape[1]), -1)]), q, out, max_rows=2000, stream=stream)
        got = out[:1].double().cpu().numpy()
        ref, bound = attention(cache, table[0], page, length, x, [length - 1], 0, "attend", type_)
        check(got, ref, bound, "tiles")
        assert rel(got, ref) < 2.0**-11 * (1 if type_ == "float16" else 8)
    pages.close()


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (3, 1, 64), (16, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("ratio", [10, 20, 24])
def test_unimportant_positions_with_large_values(gpu, type_, heads, kv, dim, ratio):
    """Every 40th position has V scales 2^ratio times the others' and almost no
    weight: the others keep their precision, whole and cut in runs."""
    page, length = 64, 2300
    pages, cache, table = pool(gpu, [length], page, kv, dim, 5)
    k, v = kv_rows(3, len(cache.k), kv, dim), kv_rows(4, len(cache.k), kv, dim)
    far = [slot_of(table, 0, p, page) for p in range(7, length, 40)]
    k[:, :, 0], k[far, :, :] = 0.0, 0.0
    k[far, :, 0] = -60.0
    v *= 2.0**-12
    v[far] *= 2.0**ratio
    refill(gpu, pages, cache, k, v)
    x = np.random.default_rng(1).standard_normal((1, heads, dim))
    x[:, :, 0] = 8.0  # scores of -42 (-60 where the heads are 64 wide)
    q, x = to_type(gpu, x, type_)
    ref, bound = decode_reference(cache, table[0], page, length, x, type_)
    work = gpu.zeros(pages.workspace_bytes(heads), dtype=gpu.uint8, device="cuda")
    for w in (None, work):
        out = gpu.zeros_like(q)
        pages.decode(0, i32(gpu, [length]), i32(gpu, table), q, out, workspace=w, stream=gpu.cuda.current_stream())
        got = out.double().cpu().numpy()
        check(got, ref, bound, f"decode, workspace {w is not None}")
        check_whole(got, ref, type_)
    pages.close()


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (3, 1, 64), (16, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("down", [12, 20, 30, 100])
def test_a_position_that_takes_the_weight_and_holds_nothing(gpu, type_, heads, kv, dim, down):
    """One position's weight is about 2^down times any other's and its V is
    zero: what the others add up to is small and as exact as ever."""
    page, length = 64, 700
    pages, cache, table = pool(gpu, [length], page, kv, dim, 5)
    k, v = np.zeros((len(cache.k), kv, dim)), kv_rows(4, len(cache.k), kv, dim)
    sink = slot_of(table, 0, 130, page)
    k[:, :, 40] = np.random.default_rng(2).standard_normal((len(k), kv)) / 50  # a factor of 2 or so between weights
    k[sink, :, :], v[sink] = 0.0, 0.0
    k[sink, :, 0] = 8.0
    refill(gpu, pages, cache, k.astype(np.float32), v)
    x = np.zeros((1, heads, dim))
    x[:, :, 0] = (down + 0.3) * np.log(2) / 8 * dim**0.5
    x[:, :, 40] = 30.0
    q, x = to_type(gpu, x, type_)
    ref, bound = decode_reference(cache, table[0], page, length, x, type_)
    assert 0 < np.abs(ref).max() < 2.0**-down * length * 8
    out = gpu.zeros_like(q)
    pages.decode(0, i32(gpu, [length]), i32(gpu, table), q, out, stream=gpu.cuda.current_stream())
    got = out.double().cpu().numpy()
    check(got, ref, bound, "decode")
    check_whole(got, ref, type_)
    pages.close()


@pytest.mark.parametrize("type_", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("down", [12, 16, 19])
def test_tiles_keep_small_weights(gpu, type_, dim, down):
    """Tiles of rows, one position with about 2^down times any other's weight
    and V of zero: the weights of the others (down to 2^-21 of the largest) have
    all of fp16's bits (2^-11), as V has, so the whole is off by their roundings and the output's alone."""
    page, length, heads, kv = 64, 700, 4, 2
    pages, cache, table = pool(gpu, [length], page, kv, dim, 5)
    k, v = np.zeros((len(cache.k), kv, dim)), 256 * kv_rows(4, len(cache.k), kv, dim)
    sink = slot_of(table, 0, 130, page)
    k[:, :, 40] = np.random.default_rng(2).standard_normal((len(k), kv)) / 50
    k[sink, :, :], v[sink] = 0.0, 0.0
    k[sink, :, 0] = 8.0
    refill(gpu, pages, cache, k.astype(np.float32), v)
    x = np.zeros((1, heads, dim))
    x[:, :, 0] = (down + 0.3) * np.log(2) / 8 * dim**0.5
    x[:, :, 40] = 30.0
    q, x = to_type(gpu, x, type_)
    q = gpu.cat([q, q.new_zeros(2000, heads, dim)])
    out, n, t = gpu.zeros_like(q), 64, i32(gpu, table)
    pages.attend(0, i32(gpu, [0] + [1] * n), i32(gpu, [length] + [0] * (n - 1)),
                 gpu.cat([t, t.new_full((n - 1, t.shape[1]), -1)]), q, out, max_rows=2000, stream=gpu.cuda.current_stream())
    got = out[:1].double().cpu().numpy()
    ref, _ = attention(cache, table[0], page, length, x, [length - 1], 0, "attend", type_)
    # three roundings, each 1 / sqrt(3) of its half step in the mean square
    off = np.linalg.norm(got - ref)
    three = ((HALF_STEP[type_]**2 + 2 * 2.0**-22) / 3)**0.5
    assert off < three * np.linalg.norm(ref) + LEAST[type_] * ref.size**0.5, (rel(got, ref), np.abs(ref).max())
    pages.close()

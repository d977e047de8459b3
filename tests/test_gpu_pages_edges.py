"""The paged cache at the edges of its tables, its scales and its queries."""
import numpy as np
import pytest

from _pages import attention, check, i32, kv_rows, pool, to_type

pytestmark = pytest.mark.gpu


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

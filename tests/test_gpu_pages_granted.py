"""Steps behind a plan that refuses: entries that did not grow keep what they
hold, bit for bit, and their rows are zeros."""
import numpy as np
import pytest

from _pages import Cache, attention, check, i32, kv_rows, slot_of, to_type
from bmo_jetson_amd import KVPages, RingError

pytestmark = pytest.mark.gpu

PAGE, LAYERS = 32, 2


class Pool:
    """Entries of the given lengths in a pool without a free page, every slot
    of every layer written; what the slots hold, in 64 bits."""

    def __init__(self, gpu, lens, width, kv, dim, seed):
        self.gpu, self.kv, self.dim = gpu, kv, dim
        need = [-(-n // PAGE) for n in lens]
        n_pages = sum(need)
        ids = iter(np.random.default_rng(seed).permutation(n_pages))
        self.host_table = [[int(next(ids)) if c < n else -1 for c in range(width)] for n in need]
        self.pages = KVPages(LAYERS, n_pages, PAGE, kv, dim)
        self.lens, self.table = i32(gpu, lens), i32(gpu, self.host_table)
        self.free = i32(gpu, np.zeros(n_pages + 2))
        self.cache = [Cache(n_pages * PAGE, kv, dim) for _ in range(LAYERS)]
        self.every = np.arange(n_pages * PAGE)
        for layer in range(LAYERS):
            k, v = (kv_rows(seed + 10 * layer + i, len(self.every), kv, dim) for i in (1, 2))
            self.cache[layer].put(self.every, k, v)
            self.pages.append(layer, i32(gpu, self.every), *(gpu.from_numpy(x).cuda() for x in (k, v)),
                              stream=gpu.cuda.current_stream())

    def check_slots(self, what):
        for layer in range(LAYERS):
            got = [self.gpu.zeros(len(self.every), self.kv, self.dim, device="cuda") for _ in range(2)]
            self.pages.gather(layer, i32(self.gpu, self.every), *got, stream=self.gpu.cuda.current_stream())
            for g, want in zip(got, (self.cache[layer].k, self.cache[layer].v)):
                assert np.array_equal(g.cpu().numpy(), want), f"{what}: layer {layer}"


@pytest.mark.parametrize("heads,kv,dim,type_", [(4, 2, 128, "bfloat16"), (3, 3, 64, "float32"), (16, 1, 128, "float16"),
                                                (16, 1, 64, "float32")])
@pytest.mark.parametrize("width", [2, 80])  # short entries; a table so wide that they can be cut in runs
def test_a_captured_step_of_entries_that_do_not_grow(gpu, heads, kv, dim, type_, width):
    """0 needs a page and finds none, 1 grows within its page, 2 pauses, 3 is
    not live, 4 fills its table; then 2 ends and 0 tries again."""
    lens = [32, 5, 20, 0, width * PAGE]
    n = len(lens)
    s = Pool(gpu, lens, width, kv, dim, 7)
    new, status = i32(gpu, [1, 1, 0, 0, 1]), i32(gpu, np.full(n, -1))
    rows = [gpu.zeros(n, heads + 2 * kv, dim, dtype=getattr(gpu, type_), device="cuda") for _ in range(LAYERS)]
    outs = [gpu.zeros(n, heads, dim, dtype=rows[0].dtype, device="cuda") for _ in range(LAYERS)]
    work = gpu.zeros(s.pages.workspace_bytes(heads), dtype=gpu.uint8, device="cuda")
    graph, side = gpu.cuda.CUDAGraph(), gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side), gpu.cuda.graph(graph, stream=side):
        stream = gpu.cuda.current_stream()
        s.pages.plan(s.free, new, s.lens, s.table, status=status, stream=stream)
        for layer in range(LAYERS):
            q, k, v = rows[layer].split([heads, kv, kv], dim=1)
            s.pages.append_decode(layer, s.lens, s.table, q, k, v, outs[layer], workspace=work, stream=stream, n_new=new,
                                  status=status)
    gpu.cuda.current_stream().wait_stream(side)
    for step in range(6):
        if step == 4:  # the paused request ends
            s.pages.plan(s.free, i32(gpu, [0, 0, -20, 0, 0]), s.lens, s.table, stream=gpu.cuda.current_stream())
            s.host_table[0][1], lens[2] = s.host_table[2][0], 0
        states = [1 if step < 4 else 0, 0, 0, 0, 2]
        grew = [b for b in (0, 1) if states[b] == 0]
        for b in grew:
            lens[b] += 1
        held = []
        for layer in range(LAYERS):
            x = np.concatenate([np.random.default_rng(100 * step + layer).standard_normal((n, heads, dim)),
                                kv_rows(100 * step + 50 + layer, n, 2 * kv, dim)], axis=1)
            t, x = to_type(gpu, x, type_)
            rows[layer].copy_(t)
            held.append(x)
            at = [slot_of(s.host_table, b, lens[b] - 1, PAGE) for b in grew]
            s.cache[layer].put(at, x[grew, heads:heads + kv], x[grew, heads + kv:])
            outs[layer].fill_(7.0)
        graph.replay()
        gpu.cuda.synchronize()
        assert status.tolist() == states and s.lens.tolist() == lens
        s.check_slots(f"step {step}")
        for layer in range(LAYERS):
            got = outs[layer].double().cpu().numpy()
            for b in range(n):
                if b not in grew:
                    assert not got[b].any(), f"step {step}, entry {b}"
                    continue
                ref, bound = attention(s.cache[layer], s.host_table[b], PAGE, lens[b], held[layer][b:b + 1, :heads],
                                       [lens[b] - 1], 0, "decode", type_)
                check(got[b:b + 1], ref, bound, f"step {step}, entry {b}, layer {layer}")
    s.pages.close()


def test_granted_refusals(gpu):
    s = Pool(gpu, [4, 4], 2, 2, 64, 1)
    q, k, two = gpu.zeros(2, 4, 64, device="cuda"), gpu.zeros(2, 2, 64, device="cuda"), i32(gpu, [0, 0])
    call = lambda **kw: s.pages.append_decode(0, s.lens, s.table, q, k, k, q.clone(), **kw)
    for kw in ({"n_new": two}, {"status": two}):
        with pytest.raises(ValueError, match="together"):
            call(**kw)
    for bad in (two[:1], two.long(), two.cpu()):
        with pytest.raises(ValueError):
            call(n_new=two, status=bad)
        with pytest.raises(ValueError):
            call(n_new=bad, status=two)
    with pytest.raises(RingError, match="layer"):
        s.pages.append_decode(LAYERS, s.lens, s.table, q, k, k, q.clone(), n_new=two, status=two)
    from bmo_jetson_amd import lib
    P = lambda t: t.data_ptr()
    for n_new, status in ((None, P(two)), (P(two), None)):
        assert lib().bmo_kv_pages_append_decode_granted(s.pages.handle, 0, 2, n_new, status, P(s.lens), P(s.table), 2, 4, 0,
                                                        P(q), 0, P(k), P(k), 0, P(q), 0.0, 0, 0, None, 0, None) == 1
    assert "null" in s.pages.last_error()
    assert lib().bmo_kv_pages_append_decode_granted(None, 0, 1, None, None, None, None, 1, 1, 0, None, 0, None, None, 0,
                                                    None, 0.0, 0, 0, None, 0, None) == 1
    call(n_new=two, status=two)
    gpu.cuda.synchronize()
    s.check_slots("nothing granted")
    s.pages.close()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dim,type_", [(64, "float16"), (128, "bfloat16")])
def test_chunks_of_which_a_plan_refuses_some(gpu, tiles, dim, type_):
    """A step of prompt pieces into a pool that runs out: refused entries' rows
    are zeros, the others' what they are among themselves, and nothing that was
    there is overwritten."""
    heads, kv, width, more = 4, 2, 3, 250
    lens = [32, 40, 20, 3, 90] + [0] * (59 if tiles else 0)  # (many entries: tiles of rows)
    n = len(lens)
    s = Pool(gpu, lens, width, kv, dim, 3)
    new = [1, 0, 12, 9, 40] + [0] * (n - 5)  # refused: 0 finds no page, 4 passes its table
    total = sum(new)
    start, slots, status = i32(gpu, np.zeros(n + 1)), i32(gpu, np.full(total, -1)), i32(gpu, np.full(n, -1))
    s.pages.plan(s.free, i32(gpu, new), s.lens, s.table, start, slots, status=status, stream=gpu.cuda.current_stream())
    states = [1, 0, 0, 0, 2] + [0] * (n - 5)
    assert status.tolist() == states
    x = np.concatenate([np.random.default_rng(8).standard_normal((total + more, heads, dim)),
                        kv_rows(9, total + more, 2 * kv, dim)], axis=1)
    t, x = to_type(gpu, x, type_)
    q, k, v = t.split([heads, kv, kv], dim=1)
    out = gpu.full((total + more, heads, dim), 7.0, dtype=q.dtype, device="cuda")
    most = 256 if tiles else max(new)
    if tiles:
        assert -(-most * 2 // 16) * n * kv >= max(1024, 2 * -(-most * 2 // 128) * n * kv + 1)
    s.pages.append(1, slots, k[:total], v[:total], stream=gpu.cuda.current_stream())
    s.pages.attend(1, start, s.lens, s.table, q, out, max_rows=most, status=status, stream=gpu.cuda.current_stream())
    got, at = out.double().cpu().numpy(), np.concatenate(([0], np.cumsum(new)))
    for b in range(5):
        if states[b] == 0:
            lens[b] += new[b]
            where = [slot_of(s.host_table, b, p, PAGE) for p in range(lens[b] - new[b], lens[b])]
            if where:
                s.cache[1].put(where, x[at[b]:at[b + 1], heads:heads + kv], x[at[b]:at[b + 1], heads + kv:])
    s.check_slots("chunks")
    for b in range(5):
        part = slice(at[b], at[b + 1])
        if states[b]:
            assert not got[part].any()
        elif new[b]:
            ref, bound = attention(s.cache[1], s.host_table[b], PAGE, lens[b], x[part, :heads],
                                   list(range(lens[b] - new[b], lens[b])), 0, "attend", type_)
            check(got[part], ref, bound, f"entry {b}")
    assert (got[total:] == 7.0).all()
    # cross attention likewise: a refused entry has nothing that is read
    s.pages.attend(1, start, s.lens, s.table, q, out, causal=False, max_rows=most, status=status,
                   stream=gpu.cuda.current_stream())
    assert not out[at[0]:at[1]].any() and not out[at[4]:at[5]].any() and bool(out[at[2]:at[4]].any(-1).all())
    with pytest.raises(ValueError, match="status"):
        s.pages.attend(1, start, s.lens, s.table, q, out, status=status[:-1])
    from bmo_jetson_amd import lib
    P = lambda z: z.data_ptr()
    assert lib().bmo_kv_pages_attend_granted(s.pages.handle, 0, n, None, P(start), P(s.lens), P(s.table), width, total, heads,
                                             1, P(q), 0, P(out), 0.0, 1, 0, 0, 0, None, 0, None) == 1
    assert lib().bmo_kv_pages_attend_granted(None, 0, 1, None, None, None, None, 1, 1, 1, 1, None, 0, None, 0.0, 1, 0, 0, 0,
                                             None, 0, None) == 1
    s.pages.close()

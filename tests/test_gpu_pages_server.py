"""The paged cache's operators run together as a server runs them: prompts in
chunks, steps of a token from a captured graph, drafts taken back, requests that
end and others that get their pages, and cross attention; against histories
that know no pages, in 64 bits."""
import numpy as np
import pytest

from _pages import Cache, attention, check, i32, kv_rows, to_type
from bmo_jetson_amd import KVPages

pytestmark = pytest.mark.gpu

LAYERS = 2


class History:
    """What one request has said, a Cache per layer whose slots are positions."""

    def __init__(self, kv, dim):
        self.kv, self.dim, self.k, self.v = kv, dim, [[], []], [[], []]

    def say(self, layer, k, v):
        self.k[layer] += list(k)
        self.v[layer] += list(v)

    def cut(self, n):
        for rows in self.k + self.v:
            del rows[len(rows) - n:]

    def ask(self, layer, q, last, kind, type_, window=0):
        n = len(self.k[layer])
        c = Cache(n, self.kv, self.dim)
        c.put(np.arange(n), np.array(self.k[layer]), np.array(self.v[layer]))
        return attention(c, np.arange(n), 1, n, q, last, window, kind, type_)


class Server:
    def __init__(self, gpu, entries, heads, kv, dim, page, n_pages, width, type_, window=0):
        self.gpu, self.heads, self.kv, self.dim, self.type_, self.window = gpu, heads, kv, dim, type_, window
        self.pages = KVPages(LAYERS, n_pages, page, kv, dim)
        self.free, self.lens = i32(gpu, np.zeros(n_pages + 2)), i32(gpu, np.zeros(entries))
        self.table = i32(gpu, np.full((entries, width), -1))
        self.status = i32(gpu, np.full(entries, -1))
        self.work = gpu.zeros(self.pages.workspace_bytes(heads), dtype=gpu.uint8, device="cuda")
        self.pages.list_init(self.free, stream=gpu.cuda.current_stream())
        self.said = [History(kv, dim) for _ in range(entries)]
        self.seed = 0

    def rows(self, n):
        """A packed QKV activation: (its views q, k, v; what they hold)."""
        self.seed += 1
        r = np.random.default_rng(self.seed)
        x = np.concatenate([r.standard_normal((n, self.heads, self.dim)),
                            kv_rows(self.seed + 1000, n, 2 * self.kv, self.dim)], axis=1)
        t, x = to_type(self.gpu, x, self.type_)
        cut = [0, self.heads, self.heads + self.kv, self.heads + 2 * self.kv]
        return [t[:, a:b] for a, b in zip(cut, cut[1:])], [x[:, a:b] for a, b in zip(cut, cut[1:])]

    def chunk(self, n_new, room=5):
        """Prompt pieces of n_new[b] tokens, in a batch padded by room rows."""
        gpu, stream = self.gpu, self.gpu.cuda.current_stream()
        total = int(sum(n_new))
        start = i32(gpu, np.zeros(len(n_new) + 1))
        slots = i32(gpu, np.full(total + room, -1))
        self.pages.plan(self.free, i32(gpu, n_new), self.lens, self.table, start, slots, status=self.status,
                        stream=stream)
        assert not self.status.any()
        for layer in range(LAYERS):
            (q, k, v), (xq, xk, xv) = self.rows(total + room)
            out = gpu.full((total + room, self.heads, self.dim), 3.0, dtype=q.dtype, device="cuda")
            self.pages.append(layer, slots, k, v, stream=stream)
            self.pages.attend(layer, start, self.lens, self.table, q, out, window=self.window, max_rows=max(n_new),
                              workspace=self.work, stream=stream)
            got = out.double().cpu().numpy()
            assert (got[total:] == 3.0).all()
            at = 0
            for b, n in enumerate(n_new):
                if n == 0:
                    continue
                rows = slice(at, at + n)
                self.said[b].say(layer, xk[rows], xv[rows])
                have = len(self.said[b].k[layer])
                ref, bound = self.said[b].ask(layer, xq[rows], have - n + np.arange(n), "attend", self.type_, self.window)
                check(got[rows], ref, bound, f"chunk, entry {b}, layer {layer}")
                at += n

    def give(self, n):
        """Takes n[b] tokens back (all of them: the request ends)."""
        self.pages.plan(self.free, i32(self.gpu, [-x for x in n]), self.lens, self.table, status=self.status,
                        stream=self.gpu.cuda.current_stream())
        assert not self.status.any()
        for b, x in enumerate(n):
            have = len(self.said[b].k[0])
            self.said[b].cut(min(x, have))
        assert self.lens.cpu().tolist() == [len(s.k[0]) for s in self.said]

    def stepper(self, live):
        """A step of a token for the live entries (lens counts stay 0 for the
        others) as a graph: (static inputs, outputs, replay)."""
        gpu, n = self.gpu, len(self.said)
        new = i32(gpu, [1 if b in live else 0 for b in range(n)])
        rows = [gpu.zeros(n, self.heads + 2 * self.kv, self.dim, dtype=getattr(gpu, self.type_), device="cuda")
                for _ in range(LAYERS)]
        outs = [gpu.zeros(n, self.heads, self.dim, dtype=rows[0].dtype, device="cuda") for _ in range(LAYERS)]
        graph, side = gpu.cuda.CUDAGraph(), gpu.cuda.Stream()
        side.wait_stream(gpu.cuda.current_stream())
        with gpu.cuda.stream(side), gpu.cuda.graph(graph, stream=side):
            s = gpu.cuda.current_stream()
            self.pages.plan(self.free, new, self.lens, self.table, status=self.status, stream=s)
            for layer in range(LAYERS):
                q, k, v = rows[layer].split([self.heads, self.kv, self.kv], dim=1)
                self.pages.append_decode(layer, self.lens, self.table, q, k, v, outs[layer], window=self.window,
                                         workspace=self.work, stream=s)
        gpu.cuda.current_stream().wait_stream(side)

        def step():
            held = []
            for layer in range(LAYERS):
                (q, k, v), x = self.rows(n)
                rows[layer].copy_(gpu.cat([q, k, v], dim=1))
                held.append(x)
            graph.replay()
            gpu.cuda.synchronize()
            assert not self.status.any()
            for layer in range(LAYERS):
                got, (xq, xk, xv) = outs[layer].double().cpu().numpy(), held[layer]
                for b in range(n):
                    if b not in live:
                        assert not got[b].any()
                        continue
                    self.said[b].say(layer, xk[b:b + 1], xv[b:b + 1])
                    have = len(self.said[b].k[layer])
                    ref, bound = self.said[b].ask(layer, xq[b:b + 1], [have - 1], "decode", self.type_, self.window)
                    check(got[b:b + 1], ref, bound, f"step, entry {b}, layer {layer}, {have} positions")
        step.keep = (new, rows, outs, graph)
        return step


@pytest.mark.parametrize("heads,kv,dim,page,type_,window", [
    (4, 2, 128, 16, "bfloat16", 0), (6, 1, 64, 32, "float16", 40), (16, 1, 128, 32, "bfloat16", 0),
    (2, 2, 64, 64, "float16", 0)])
def test_requests_come_and_go(gpu, heads, kv, dim, page, type_, window):
    width = -(-260 // page)
    s = Server(gpu, 4, heads, kv, dim, page, 2 * width + 6, width, type_, window)
    s.chunk([37, 0, 5, 0])
    s.chunk([60, 0, 0, 150])  # the next piece of the first, another's whole prompt
    step = s.stepper([0, 2, 3])
    for _ in range(page + 2):  # over a page's end
        step()
    s.give([3, 0, 1, 0])  # drafts refused
    for _ in range(3):
        step()
    s.give([0, 0, 0, 1000])  # the fourth ends; its pages go to the second
    s.chunk([0, 130, 1, 0])
    step.keep[0].copy_(i32(gpu, [1, 1, 1, 0]))
    step = s.stepper([0, 1, 2])
    for _ in range(2):
        step()
    s.give([1000] * 4)
    f = s.free.cpu().numpy()
    assert f[0] == s.pages.n_pages and sorted(f[2:]) == list(range(s.pages.n_pages))
    s.pages.close()


@pytest.mark.parametrize("heads,kv,dim,type_", [(4, 4, 64, "float16"), (8, 2, 128, "bfloat16")])
def test_a_decoder_reads_its_encoders_states(gpu, heads, kv, dim, type_):
    """Encoders' states once into the pages, then cross attention: a chunk of
    rows, and a token each."""
    s = Server(gpu, 3, heads, kv, dim, 32, 20, 7, type_)
    n_new, stream = [200, 33, 64], gpu.cuda.current_stream()
    slots = i32(gpu, np.zeros(sum(n_new)))
    s.pages.plan(s.free, i32(gpu, n_new), s.lens, s.table, slots=slots, stream=stream)
    for layer in range(LAYERS):
        (_, k, v), (_, xk, xv) = s.rows(sum(n_new))
        s.pages.append(layer, slots, k, v, stream=stream)
        at = np.concatenate(([0], np.cumsum(n_new)))
        for b in range(3):
            s.said[b].say(layer, xk[at[b]:at[b + 1]], xv[at[b]:at[b + 1]])
    for rows in ([4, 1, 7], [0, 150, 20]):
        for layer in range(LAYERS):
            (q, _, _), (xq, _, _) = s.rows(sum(rows))
            out = gpu.zeros(sum(rows), heads, dim, dtype=q.dtype, device="cuda")
            start = np.concatenate(([0], np.cumsum(rows)))
            s.pages.attend(layer, i32(gpu, start), s.lens, s.table, q, out, causal=False, max_rows=max(rows),
                           workspace=s.work, stream=stream)
            got = out.double().cpu().numpy()
            for b in range(3):
                part = slice(start[b], start[b + 1])
                ref, bound = s.said[b].ask(layer, xq[part], [n_new[b] - 1] * rows[b], "attend", type_)
                check(got[part], ref, bound, f"cross, entry {b}")
    (q, _, _), (xq, _, _) = s.rows(3)
    out = gpu.zeros(3, heads, dim, dtype=q.dtype, device="cuda")
    s.pages.decode(1, s.lens, s.table, q, out, workspace=s.work, stream=stream)
    got = out.double().cpu().numpy()
    for b in range(3):
        ref, bound = s.said[b].ask(1, xq[b:b + 1], [n_new[b] - 1], "decode", type_)
        check(got[b:b + 1], ref, bound, f"cross token, entry {b}")
    s.pages.close()


def test_a_small_workspace_cuts_less(gpu):
    """Any size is taken; what does not fit is not cut, and nothing is written
    behind the end."""
    s = Server(gpu, 2, 4, 2, 128, 64, 100, 45, "float16")
    s.chunk([2800, 40])
    (q, _, _), (xq, _, _) = s.rows(2)
    full = s.pages.workspace_bytes(4)
    for size in (16, 8000, 40000, full // 7 // 16 * 16, full):
        guard = gpu.full((full // 4 + 1024,), 5.0, device="cuda")
        for attend in (False, True):
            out = gpu.zeros(2, 4, 128, dtype=q.dtype, device="cuda")
            kw = dict(workspace=guard[:size // 4], stream=gpu.cuda.current_stream())
            if attend:
                s.pages.attend(1, i32(gpu, [0, 1, 2]), s.lens, s.table, q, out, max_rows=1, **kw)
            else:
                s.pages.decode(1, s.lens, s.table, q, out, **kw)
            got = out.double().cpu().numpy()
            for b, n in enumerate((2800, 40)):
                ref, bound = s.said[b].ask(1, xq[b:b + 1], [n - 1], "decode", "float16")
                check(got[b:b + 1], ref, bound, f"{size} bytes, entry {b}")
            assert bool((guard[size // 4:] == 5.0).all())
    s.pages.close()


@pytest.mark.parametrize("dim,heads", [(128, 16), (64, 16)])
def test_pages_past_32_bits_of_bytes(gpu, dim, heads):
    """The last pages of a pool of 5 GB give the bits that the first ones of a
    small pool give, in every kernel."""
    kv, page, lens, stream = 8, 1024, [1500, 90], gpu.cuda.current_stream()
    n_pages = 5 * 2**30 // (kv * page * dim * 36 // 32)
    rows = sum(lens)
    k, v = gpu.randn(rows, kv, dim, device="cuda"), gpu.randn(rows, kv, dim, device="cuda")
    new = gpu.randn(2, heads + 2 * kv, dim, device="cuda")
    results = []
    for pages, first in ((KVPages(1, 4, page, kv, dim), 0), (KVPages(1, n_pages, page, kv, dim), n_pages - 3)):
        table = np.array([[first + 2, first], [first + 1, -1]])
        pos = np.concatenate([np.arange(n) for n in lens])
        entry = np.repeat([0, 1], lens)
        slots = table[entry, pos // page] * page + pos % page
        table = i32(gpu, table)
        pages.append(0, i32(gpu, slots), k, v, stream=stream)
        got = []
        for type_ in ("float32", "bfloat16"):
            q = new[:, :heads].to(getattr(gpu, type_))
            out = gpu.zeros_like(q)
            pages.decode(0, i32(gpu, lens), table, q, out, stream=stream)
            got.append(out)
        x = new.half()
        out = gpu.zeros(2, heads, dim, dtype=gpu.half, device="cuda")
        pages.append_decode(0, i32(gpu, [n + 1 for n in lens]), table, x[:, :heads], x[:, heads:heads + kv],
                            x[:, heads + kv:], out, stream=stream)
        got.append(out)
        back = [gpu.zeros(rows, kv, dim, device="cuda") for _ in range(2)]
        pages.gather(0, i32(gpu, slots), *back, stream=stream)
        got += back
        q = new[:, :heads].repeat(40, 1, 1).bfloat16()
        for batch in (2, 130):  # sets of columns, tiles
            start = i32(gpu, [0, 40] + [80] * (batch - 1))
            many = gpu.cat([table, table.new_full((batch - 2, 2), -1)])
            out = gpu.zeros_like(q)
            pages.attend(0, start, i32(gpu, lens + [0] * (batch - 2)), many, q, out, max_rows=40 if batch == 2 else 256,
                         stream=stream)
            got.append(out)
        results.append([x.cpu() for x in got])
        pages.close()
    for a, b in zip(*results):
        assert gpu.equal(a, b) and bool(a.any())

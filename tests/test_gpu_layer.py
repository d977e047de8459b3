"""A transformer layer of a server's step from the operators together: norm,
projections, rotary positions, the paged cache's attention, gated feed-forward,
as one captured step over entries of different lengths, against 64 bits."""
import math

import numpy as np
import pytest

from _pages import attention, Cache, q4_0 as quantized, rel
from _rows import blocks_of, q4_0, split8, values8

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE = 8, 2, 64, 32
WIDTH, HIDDEN = HEADS * DIM, 736


def _model(seed):
    out = {}
    for i, (name, rows, cols) in enumerate((("qkv", (HEADS + 2 * KV) * DIM, WIDTH), ("out", WIDTH, WIDTH),
                                            ("in", 2 * HIDDEN, WIDTH), ("down", WIDTH, HIDDEN))):
        _, codes, scales = q4_0(seed + i, rows, cols)
        scales = np.abs(scales)
        out[name] = (blocks_of(codes, scales), ((codes.astype(np.float64) - 8) * scales.astype(np.float64)[:, :, None])
                     .reshape(rows, cols))
    r = np.random.default_rng(seed)
    for name in ("w1", "w2"):
        out[name] = r.uniform(0.5, 1.5, WIDTH).astype(np.float32)
    return out


class Plain:
    """The layer in 64 bits; rows pass through 8 bits as the library's do."""

    def __init__(self, model, n_slots):
        self.m, self.cache = model, Cache(n_slots, KV, DIM)

    def norm(self, h, w):
        y = h / np.sqrt((h * h).mean(axis=1, keepdims=True) + 1e-5) * w
        return values8(*split8(y.astype(np.float32)))

    def step(self, x, res, pos, slots, tables, lens):
        res = res + x
        packed = (self.norm(res, self.m["w1"]) @ self.m["qkv"][1].T).reshape(len(x), -1, DIM)
        angle = pos[:, None] * 10000.0 ** (-2.0 * np.arange(DIM // 2) / DIM)
        turn = np.exp(1j * angle)[:, None, :]
        qk = packed[:, :HEADS + KV].reshape(len(x), HEADS + KV, DIM // 2, 2)
        z = (qk[..., 0] + 1j * qk[..., 1]) * turn
        qk = np.stack((z.real, z.imag), axis=3).reshape(len(x), HEADS + KV, DIM)
        self.cache.put(slots, qk[:, HEADS:].astype(np.float32), packed[:, HEADS + KV:].astype(np.float32))
        att = np.concatenate([attention(self.cache, tables[b], PAGE, lens[b], qk[b:b + 1, :HEADS], [lens[b] - 1], 0, "decode",
                                        "float32")[0] for b in range(len(x))])
        res = res + values8(*split8(att.reshape(len(x), WIDTH).astype(np.float32))) @ self.m["out"][1].T
        both = self.norm(res, self.m["w2"]) @ self.m["in"][1].T
        g, u = both[:, :HIDDEN], both[:, HIDDEN:]
        h = g / (1 + np.exp(-g)) * u
        return values8(*split8(h.astype(np.float32))) @ self.m["down"][1].T, res


@pytest.mark.parametrize("n", [1, 5, 40])
def test_steps_of_a_layer(gpu, n):
    torch = gpu
    from bmo_jetson_amd import KVPages, Q4Weights, Rope, quantize_rows, rms_norm
    model = _model(3)
    weights = {}
    for name in ("qkv", "out", "in", "down"):
        b = model[name][0]
        weights[name] = Q4Weights(b.shape[0], b.shape[1] * 32)
        weights[name].load(torch.from_numpy(b).cuda(), stream=torch.cuda.current_stream())
    w1, w2 = (torch.from_numpy(model[k]).cuda() for k in ("w1", "w2"))
    rope = Rope(DIM)
    steps = 5
    n_pages = n * 2 + 1
    pages = KVPages(1, n_pages, PAGE, KV, DIM)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    f32 = lambda *s: torch.zeros(*s, device="cuda")
    rows8 = lambda cols: (torch.zeros(n, cols, dtype=torch.int8, device="cuda"),
                          torch.zeros(n, cols // 32, dtype=torch.float16, device="cuda"))
    free, table, lens, new, status = i32(n_pages + 2), i32(n, 2), i32(n), i32(n) + 1, i32(n)
    start, slots, positions, entries = i32(n + 1), i32(n), i32(n), i32(n)
    x, res, packed, att = f32(n, WIDTH), f32(n, WIDTH), f32(n, HEADS + 2 * KV, DIM), f32(n, HEADS, DIM)
    (c, s), (hc, hs) = rows8(WIDTH), rows8(HIDDEN)
    q, k, v = packed[:, :HEADS], packed[:, HEADS:HEADS + KV], packed[:, HEADS + KV:]
    k_dense, v_dense = f32(n, KV, DIM), f32(n, KV, DIM)
    pages.list_init(free, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()

    def step():
        st = torch.cuda.current_stream()
        pages.plan(free, new, lens, table, start, slots, positions, entries, status, stream=st)
        rms_norm(x, w1, residual=res, codes=c, scales=s, stream=st)
        weights["qkv"].product(c, s, packed.view(n, -1), stream=st)
        rope.apply(positions, q, k, stream=st)
        pages.append_decode(0, lens, table, q, k, v, att, n_new=new, status=status, stream=st)
        quantize_rows(att.view(n, WIDTH), c, s, stream=st)
        weights["out"].product(c, s, x, stream=st)
        rms_norm(x, w2, residual=res, codes=c, scales=s, stream=st)
        weights["in"].gated(c, s, hc, hs, stream=st)
        weights["down"].product(hc, hs, x, stream=st)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    plain = Plain(model, n_pages * PAGE)
    for t in range(steps):
        x0 = np.random.default_rng(100 + t).standard_normal((n, WIDTH)).astype(np.float32)
        x.copy_(torch.from_numpy(x0))
        res.zero_()
        if t == 0:
            step()  # eager
        else:
            graph.replay()
        torch.cuda.synchronize()
        want, want_res = plain.step(x0.astype(np.float64), np.zeros((n, WIDTH)), positions.cpu().numpy(), slots.cpu().numpy(),
                                    table.cpu().numpy(), lens.cpu().numpy())
        assert (positions == t).all() and (status == 0).all()
        # Both round rows to 8 bits and keys and values to 4.  A value within fp32's noise (some 1e-6 of its block's
        # largest) of the middle between two codes takes the other one, in a share 127 * 2e-6 of the codes (4 bits:
        # 8 * 2e-6), off by one step, 1 / 127 (1 / 8) of its block's largest, some 3 times the norm's root: at most
        # sqrt(3e-4) / 40 = 4e-4 and sqrt(2e-5) * 3 / 8 = 2e-3 of a row's norm, passed on through the products and, by
        # the scores, magnified by their size (up to 4 here).
        assert rel(x.cpu().numpy(), want) < 0.01 and rel(res.cpu().numpy(), want_res) < 0.01, t

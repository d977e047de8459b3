"""Test helper: the paged cache's operators written out plainly, in 64 bits.

Bounds (per output, from the kernels' arithmetic):

decode   fp32: a weight enters as two fp16 parts (2^-21 of itself, were the
         parts truncated; they are rounded, 2^-22), codes are exact, sums are fp32 (some hundred roundings of 2^-24 of at
         most 8 sum p|d|): 2^-16 * 16 sum p|d| covers both; a score is off by at
         most 2^-21 max|q| sum|k| (half a step of a query of 22 bits, the step
         being at most 2^-20 of the row's largest; it has 23) in log2 units, which moves a
         weight and the sum by ln 2 of that each.  16 bits: a weight rounds to
         fp16, 2^-11 of sum p|v|, and the query has 15 bits, 2^-14 there.
attend   V and the weights round to fp16 (2^-11 each; a weight below 2^-14 is
         off by 2^-25 of the largest instead), K too, which moves a score by
         2^-11 sum|q k|, a weight and the sum by ln 2 of that each.
Both then round once to the output's type, half a step: 2^-8 (bf16), 2^-11
(fp16), 2^-24 (fp32) of the value."""
from __future__ import annotations

import math

import numpy as np

import oracle

HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
LN2 = math.log(2.0)


def q4_0(x):
    """(values in 64 bits, scales) of fp32 rows [...][dim] as Q4_0."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    blocks = oracle.quantize_q4_0(x.reshape(-1))
    v = oracle.dequantize_q4_0(blocks).astype(np.float64).reshape(x.shape)
    d = np.frombuffer(np.ascontiguousarray(blocks).tobytes(), dtype=np.uint8).reshape(-1, 18)[:, :2].copy()
    return v, d.view(np.float16).astype(np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32)


class Cache:
    """What a pool's slots hold: values of K and V and V's scales, per slot."""

    def __init__(self, n_slots, kv, dim):
        self.k = np.zeros((n_slots, kv, dim))
        self.v = np.zeros((n_slots, kv, dim))
        self.d = np.zeros((n_slots, kv, dim // 32))

    def put(self, slots, k, v):
        slots = np.asarray(slots)
        real = (slots >= 0) & (slots < len(self.k))
        self.k[slots[real]] = q4_0(k[real])[0]
        self.v[slots[real]], self.d[slots[real]] = q4_0(v[real])


def attention(cache, table_row, page, length, q, last, window, kind, type_, scale=None):
    """Rows q [n][heads][dim] (64 bits) of one entry, row i seeing positions
    up to last[i], no more than window of them (0: all): (out, bound)."""
    n, heads, dim = q.shape
    kv = cache.k.shape[1]
    n_pages = len(cache.k) // page
    scale = dim**-0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    pos = np.arange(min(max(length, 0), len(table_row) * page))
    ids = np.asarray(table_row)[pos // page]
    good = (ids >= 0) & (ids < n_pages)
    slots = np.where(good, ids * page + pos % page, 0)
    for i in range(n):
        seen = good & (pos <= last[i])
        if window:
            seen &= pos > last[i] - window
        if not seen.any():
            continue
        s = slots[seen]
        for h in range(heads):
            g = h // (heads // kv)
            k, v, d = cache.k[s, g], cache.v[s, g], np.repeat(np.abs(cache.d[s, g]), 32, axis=1)
            score = k @ q[i, h] * scale
            p = np.exp(score - score.max())
            p /= p.sum()
            o = p @ v
            out[i, h] = o
            if kind == "decode":
                full = type_ == "float32"
                off = 2.0**(-21 if full else -14) * np.abs(q[i, h]).max() * np.abs(k).sum(axis=1).max() * scale / LN2
                b = 2.0**-16 * 16 * (p @ d) + (2 * LN2 * off + (0 if full else 2.0**-11)) * (p @ np.abs(v))
            else:
                off = 2.0**-11 * (np.abs(k) @ np.abs(q[i, h])).max() * scale / LN2
                b = (2 * 2.0**-11 + 2 * LN2 * off) * (p @ np.abs(v)) + 2.0**-25 * np.abs(v).sum(axis=0)
            bound[i, h] = b + HALF_STEP[type_] * (np.abs(o) + b)
    return out, bound


def check(got, ref, bound, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert np.all(np.isfinite(got)), f"{what}: not finite"
    over = np.abs(got - ref) > bound + 1e-30
    assert not over.any(), (f"{what}: {over.sum()} of {over.size} past the bound, first at {np.argwhere(over)[0]}, "
                            f"largest {np.abs(got - ref).max():.3e}, norm {rel(got, ref):.3e}")


def rel(got, ref):
    return float(np.linalg.norm(np.asarray(got, dtype=np.float64) - ref) / max(np.linalg.norm(ref), 1e-300))


def kv_rows(seed, *shape):
    """N(0, 1), one element in a hundred 8 times as large."""
    r = np.random.default_rng(seed)
    x = r.standard_normal(shape)
    return np.where(r.random(shape) < 0.01, 8 * x, x).astype(np.float32)


def to_type(torch, x, type_):
    """x as a tensor of the type on the GPU, and what it holds in 64 bits."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, type_))
    return t.cuda(), t.double().numpy()


def i32(torch, x):
    return torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


def pool(torch, lens, page, kv, dim, seed, layers=1, layer=0, spare=2):
    """A pool with every slot written and a table of the lengths, pages dealt
    out at random: (pages, cache, table)."""
    from bmo_jetson_amd import KVPages
    need = [-(-max(n, 0) // page) for n in lens]
    n_pages = sum(need) + spare
    ids = np.random.default_rng(seed).permutation(n_pages)
    table = np.full((len(lens), max(1, max(need))), -1, dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    pages = KVPages(layers, n_pages, page, kv, dim)
    cache = Cache(n_pages * page, kv, dim)
    slots = np.arange(n_pages * page)
    k, v = kv_rows(seed + 1, len(slots), kv, dim), kv_rows(seed + 2, len(slots), kv, dim)
    cache.put(slots, k, v)
    pages.append(layer, i32(torch, slots), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(),
                 stream=torch.cuda.current_stream())
    return pages, cache, table


def slot_of(table, b, pos, page):
    return int(table[b][pos // page]) * page + pos % page

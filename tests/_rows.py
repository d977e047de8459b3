"""Test helper: the operators on rows written out plainly, in 64 bits, with the
bounds that their arithmetic in 32 bits allows (U is half a step of fp32)."""
from __future__ import annotations

import numpy as np

U = 2.0**-24
HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
# half a step of the smallest subnormals
TINY = {"float32": 2.0**-150, "float16": 2.0**-25, "bfloat16": 2.0**-134}


def rounded(bound, ref, type_):
    """A bound of values in 32 bits, after their rounding to the type."""
    return bound + HALF_STEP[type_] * (np.abs(ref) + bound) + TINY[type_]


def tensor(torch, x, type_, device="cuda"):
    """x as a tensor of the type, and what it holds in 64 bits."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, type_))
    return t.to(device), t.double().numpy()


def check(got, ref, bound, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    both = np.isnan(got) & np.isnan(ref) | (got == ref)
    with np.errstate(invalid="ignore"):
        over = ~(np.abs(got - ref) <= bound) & ~both
    assert not over.any(), (f"{what}: {over.sum()} of {over.size} past the bound, first at {np.argwhere(over)[0]}: "
                            f"{got[tuple(np.argwhere(over)[0])]} for {ref[tuple(np.argwhere(over)[0])]}")


def scale8(amax):
    """The least fp16 that is not below amax (fp32) / 127; NaN where there is none."""
    amax = np.asarray(amax, dtype=np.float32).astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        h = (amax / 127).astype(np.float16)
        up = np.nextafter(h, np.float16(np.inf))
        h = np.where(h.astype(np.float64) * 127 < amax, up, h)  # (18 bits: exact)
        return np.where(np.isfinite(h), h, np.float16(np.nan)).astype(np.float16)


def split8(x):
    """fp32 rows as (codes, scales) by the definition."""
    b = np.asarray(x, dtype=np.float32).reshape(x.shape[0], -1, 32)
    d = scale8(np.abs(b).max(axis=2))
    s = d.astype(np.float64)[:, :, None]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(s > 0, np.rint(b.astype(np.float64) / s), 0.0)
    return q.astype(np.int8).reshape(x.shape), d


def values8(codes, scales):
    n = codes.shape[0]
    return (codes.astype(np.float64).reshape(n, -1, 32) * scales.astype(np.float64)[:, :, None]).reshape(n, -1)


def check8(codes, scales, ref, off, what=""):
    """8-bit rows of values that are within `off` of ref (64 bits): a code is
    the integer nearest to its value / scale, the scale the least that fits."""
    codes, d = np.asarray(codes), np.asarray(scales).astype(np.float64)
    n = codes.shape[0]
    v, e, q = (a.reshape(n, -1, 32) for a in (ref, np.broadcast_to(off, ref.shape), codes.astype(np.float64)))
    lost = ~np.isfinite(v).all(axis=2) | (np.abs(v).max(axis=2) > 127 * 65504.0)
    assert np.array_equal(np.isnan(d), lost), f"{what}: NaN scales at {np.argwhere(np.isnan(d) != lost)[:3]}"
    assert not q[lost].any(), what
    v, e, q, d = v[~lost], e[~lost], q[~lost], d[~lost]
    assert (np.abs(q) <= 127).all(), what
    lo, hi = (np.abs(v) - e).max(axis=1).clip(0), (np.abs(v) + e).max(axis=1)
    least, most = lo / 127 * (1 - 2 * U), scale8(hi.astype(np.float32) * np.float32(1 + 4 * U)).astype(np.float64)
    most = np.where(np.isnan(most), 65504.0, most)  # (a value that has a scale, whose margin has none)
    assert (d >= least).all() and (d <= most).all(), (what, np.argwhere((d < least) | (d > most))[:3])
    # (x / d as a product with 1 / d: two roundings of at most 127)
    bound = d[:, None] * (0.5 + 127 * 4 * U) + e
    over = np.abs(q * d[:, None] - v) > bound
    assert not over.any(), (what, np.argwhere(over)[:3])


def q4_0(seed, rows, cols):
    """Random Q4_0 weights: ggml blocks, and values in 64 bits."""
    r = np.random.default_rng(seed)
    codes = np.clip(np.rint(r.standard_normal((rows, cols // 32, 32)) * 3 + 8), 0, 15).astype(np.uint8)
    scales = (r.uniform(-1, 1, (rows, cols // 32)) / np.sqrt(cols)).astype(np.float16)
    return blocks_of(codes, scales), codes, scales


def blocks_of(codes, scales):
    rows, nb, _ = codes.shape
    out = np.empty((rows, nb, 18), dtype=np.uint8)
    out[:, :, :2] = np.ascontiguousarray(scales).view(np.uint8).reshape(rows, nb, 2)
    out[:, :, 2:] = codes[:, :, :16] | codes[:, :, 16:] << 4
    return out


def product(codes, scales, w_codes, w_scales):
    """(out, bound): 8-bit rows times Q4_0 weights.  A block's sum is exact, a
    part d4 * d8 * sum has one rounding, its addition one for each of the blocks
    before it and of up to 32 partial sums."""
    m, nb = scales.shape
    q = codes.astype(np.float64).reshape(m, nb, 32)
    c = w_codes.astype(np.float64) - 8
    d8, d4 = scales.astype(np.float64), w_scales.astype(np.float64)
    out, size = np.zeros((m, len(c))), np.zeros((m, len(c)))
    with np.errstate(invalid="ignore"):
        for b in range(nb):
            part = (q[:, b] @ c[:, b].T) * d8[:, b, None] * d4[None, :, b]
            out += part
            size += np.abs(part)
    return out, (nb + 34) * U * size


def gated(g, u, g_off, u_off, activation):
    """(h, bound) of act(g) * u; the activations' slopes are at most 1.13, and
    exp, the quotient and the products add some 16 roundings."""
    with np.errstate(over="ignore", invalid="ignore"):
        a = g if activation == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g**3)
        # (the argument of exp has some roundings of its own: a move of 4 U |a|, where the activation is not flat)
        f = g / (1 + np.exp(-a))
        h = f * u
        flat = np.abs(g) * np.abs(a) * np.exp(-np.abs(a)) * 8 * U
        return h, 1.13 * g_off * (np.abs(u) + u_off) + np.abs(f) * u_off + flat * np.abs(u) + np.abs(h) * 16 * U + 1e-37

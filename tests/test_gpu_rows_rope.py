"""Rotary positions against 64 bits."""
import math

import numpy as np
import pytest

from _rows import U, check, rounded, tensor

pytestmark = pytest.mark.gpu


def rates(rot, theta=10000.0, factor=1.0, trained=0, fast=32.0, slow=1.0, divisors=None):
    """Radians a position, written apart from the library's."""
    out = []
    for i in range(rot // 2):
        r = theta ** (-2.0 * i / rot)
        if trained:
            at = [rot * math.log(trained / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (fast, slow)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            t = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            r = r * (1 - t) + r / factor * t
        else:
            r /= factor
        out.append(r / (divisors[i] if divisors is not None else 1.0))
    return np.array(out)


def turned(x, pos, r, m, rot, interleaved):
    """(rows, bound): each of the two products of an output has its cosine's or
    sine's rounding and its own, their sum one."""
    angle = np.asarray(pos, dtype=np.float64)[:, None] * r
    c, s = (f(angle)[:, None, :] * m for f in (np.cos, np.sin))
    y, bound = x.copy(), np.zeros_like(x)
    t = np.s_[..., :rot]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * c - b * s, a * s + b * c
    # (and an angle of 64 bits is off by a rounding or two: 2^31 * 2^-52)
    far = np.abs(angle)[:, None, :] * 2.0**-51 * m
    size = (np.abs(a) + np.abs(b)) * (m * 3.5 * U + far)
    pair = (lambda p, q: np.stack((p, q), axis=3).reshape(x[t].shape)) if interleaved else \
        (lambda p, q: np.concatenate((p, q), axis=2))
    y[t], bound[t] = pair(u, v), pair(size, size)
    return y, bound


def _run(torch, dim, rot, interleaved, type_, n=5, heads=3, kv=2, pos=None, seed=0, **scaling):
    from bmo_jetson_amd import Rope
    r = np.random.default_rng(seed)
    pos = r.integers(0, 5000, n) if pos is None else np.asarray(pos)
    rope = Rope(dim, rot, interleaved=interleaved, **scaling)
    packed, p64 = tensor(torch, r.standard_normal((n, heads + 2 * kv, dim)), type_)
    q, k = packed[:, :heads], packed[:, heads:heads + kv]
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    q_out, k_out = (torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") for x in (q, k))
    before = packed.clone()
    stream = torch.cuda.current_stream()
    rope.apply(p, q, k if kv else None, q_out, k_out if kv else None, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(packed, before)
    m = scaling.get("magnitude", 0.0) or (0.1 * math.log(scaling["factor"]) + 1 if scaling.get("trained") else 1.0)
    table = rates(rot, scaling.get("theta", 10000.0), scaling.get("factor", 1.0), scaling.get("trained", 0),
                  scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0), scaling.get("divisors"))
    for got, ref in ((q_out, p64[:, :heads]), (k_out, p64[:, heads:heads + kv])):
        y, bound = turned(ref, pos, table, m, rot, interleaved)
        check(got.double().cpu().numpy(), y, rounded(bound, y, type_), f"{dim} {rot} {interleaved} {type_}")
        assert torch.equal(got[..., rot:].double().cpu(), torch.from_numpy(ref[..., rot:]))  # as they were
    rope.apply(p, q, k if kv else None, stream=stream)  # in place
    assert torch.equal(q, q_out) and torch.equal(k, k_out)
    assert torch.equal(packed[:, heads + kv:], before[:, heads + kv:])
    return rope


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (96, 24), (80, 40), (80, 20), (96, 48), (20, 12), (256, 64), (6, 4), (2, 2),
                                     (128, 2), (130, 126), (1024, 1024)])
def test_layouts_sizes_types(gpu, dim, rot, interleaved, type_):
    _run(gpu, dim, rot, interleaved, type_)


@pytest.mark.parametrize("n,heads,kv", [(1, 1, 0), (1, 32, 32), (33, 1, 1), (200, 32, 8), (1000, 5, 0), (3, 128, 1)])
def test_numbers_of_rows(gpu, n, heads, kv):
    _run(gpu, 64, 64, True, "float32", n, heads, kv)
    _run(gpu, 128, 128, False, "bfloat16", n, heads, kv)


@pytest.mark.parametrize("interleaved", [True, False])
def test_far_and_negative_positions(gpu, interleaved):
    pos = [0, 1, 2**31 - 1, -2**31, -1, 10**6, 123456789]
    _run(gpu, 128, 128, interleaved, "float32", len(pos), 2, 1, pos=pos)


@pytest.mark.parametrize("scaling", [
    dict(factor=4.0), dict(theta=500000.0, factor=8.0, trained=8192), dict(factor=40.0, trained=4096),
    dict(factor=40.0, trained=4096, beta_fast=16.0, beta_slow=2.0, magnitude=1.5), dict(theta=1.5, factor=2.0, trained=4),
    dict(divisors=[1.0 + 0.25 * i for i in range(32)]), dict(factor=1.0, trained=4096), dict(magnitude=0.25),
    dict(factor=8.0, trained=8192, divisors=[1.0 + 0.01 * i for i in range(32)])], ids=str)
def test_scaled_for_long_contexts(gpu, scaling):
    for type_, interleaved in (("float32", True), ("bfloat16", False)):
        _run(gpu, 64, 64, interleaved, type_, 6, pos=[0, 5, 4095, 70000, 131071, 1000000], **scaling)


def test_odd_strides_and_alignment(gpu):
    torch = gpu
    from bmo_jetson_amd import Rope
    rope = Rope(64, 32, interleaved=False)
    for type_ in (torch.float32, torch.bfloat16):
        base = torch.randn(4, 3 * 64 + 5, device="cuda").to(type_)
        q = base.as_strided((4, 3, 64), (3 * 64 + 5, 64, 1), 1)
        p = torch.tensor([3, 1, 4, 1], dtype=torch.int32, device="cuda")
        dense = torch.empty(4, 3, 64, dtype=type_, device="cuda")
        rope.apply(p, q, q_out=dense, stream=torch.cuda.current_stream())
        again = torch.empty_like(dense)
        rope.apply(p, q.contiguous(), q_out=again, stream=torch.cuda.current_stream())
        assert torch.equal(dense, again)
        before = base.clone()
        rope.apply(p, q, stream=torch.cuda.current_stream())
        assert torch.equal(q, dense)
        assert torch.equal(base[:, 0], before[:, 0]) and torch.equal(base[:, 193:], before[:, 193:])


def test_no_tokens_and_the_ring_s_rotation(gpu):
    """The same turns as the ring's fused rotation: keys that it appends."""
    torch = gpu
    from bmo_jetson_amd import KVRing, Rope
    rope = Rope(128)
    rope.apply(torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, 4, 128, device="cuda"))
    ring, plain = KVRing(1, 1, 4, 128, 64), KVRing(1, 1, 4, 128, 64)
    stream = torch.cuda.current_stream()
    for pos in (0, 7, 60, 63):
        q, k, v = (torch.randn(1, 4, 128, device="cuda") for _ in range(3))
        out, out2 = torch.empty_like(q), torch.empty_like(q)
        p = torch.tensor([pos], dtype=torch.int32, device="cuda")
        ring.append_decode(0, p, q, k, v, out, 4, stream=stream, rope_theta=10000.0)
        rope.apply(p, q, k, stream=stream)
        plain.append_decode(0, p, q, k, v, out2, 4, stream=stream)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(ring.export_q4_0(0, 0, 0, pos, 1), plain.export_q4_0(0, 0, 0, pos, 1))
        assert torch.equal(out, out2)


def test_captured(gpu):
    torch = gpu
    from bmo_jetson_amd import Rope
    rope = Rope(64)
    q, k = torch.randn(7, 4, 64, device="cuda"), torch.randn(7, 2, 64, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    p = torch.arange(7, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.apply(p, q, k, q_out, k_out, stream=torch.cuda.current_stream())
    for _ in range(4):
        p += 1000
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        again = torch.empty_like(q)
        rope.apply(p, q, q_out=again, stream=torch.cuda.current_stream())
        assert torch.equal(again, q_out)

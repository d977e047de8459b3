"""Rows into the paged cache's slots and back: bit-exact with the oracle's
quantizer, for every type, stride and slot order."""
import numpy as np
import pytest

import oracle
from _pages import i32, kv_rows, to_type
from bmo_jetson_amd import KVPages, KVRing, RingError

pytestmark = pytest.mark.gpu


def _blocks(x):
    x = np.ascontiguousarray(x, dtype=np.float32)
    return np.ascontiguousarray(oracle.quantize_q4_0(x.reshape(-1))).view(np.uint8).reshape(
        *x.shape[:-1], x.shape[-1] // 32, 18)


def _gathered(gpu, pages, layer, slots, type_="uint8"):
    n, kv, d = len(slots), pages.n_kv_heads, pages.head_dim
    shape = (n, kv, d // 32, 18) if type_ == "uint8" else (n, kv, d)
    k, v = (gpu.zeros(shape, dtype=getattr(gpu, type_), device="cuda") for _ in range(2))
    pages.gather(layer, i32(gpu, slots), k, v, stream=gpu.cuda.current_stream())
    return k.cpu(), v.cpu()


@pytest.mark.parametrize("dim,page,kv", [(128, 16, 1), (128, 64, 5), (64, 32, 3), (64, 128, 2), (128, 1024, 2)])
@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n", [1, 7, 100])
def test_rows_are_bit_exact(gpu, dim, page, kv, type_, n):
    n_pages = -(-150 // page) + 1
    pages = KVPages(2, n_pages, page, kv, dim)
    slots = np.random.default_rng(n).permutation(n_pages * page)[:n]
    (k, kx), (v, vx) = (to_type(gpu, kv_rows(s, n, kv, dim), type_) for s in (1, 2))
    pages.append(1, i32(gpu, slots), k, v, stream=gpu.cuda.current_stream())
    gk, gv = _gathered(gpu, pages, 1, slots)
    assert np.array_equal(gk.numpy(), _blocks(kx)) and np.array_equal(gv.numpy(), _blocks(vx))
    # every other slot, and the other layer, hold ggml's zero block
    every = np.arange(n_pages * page)
    for layer in (0, 1):
        for got in _gathered(gpu, pages, layer, every):
            got = got.numpy()[every if layer == 0 else np.setdiff1d(every, slots)]
            assert not got.any()
    # and as values, rounded once
    for out_type in ("float32", "float16", "bfloat16"):
        for got, x in zip(_gathered(gpu, pages, 1, slots, out_type), (kx, vx)):
            want = oracle.dequantize_q4_0(oracle.quantize_q4_0(x.astype(np.float32).reshape(-1))).reshape(x.shape)
            assert gpu.equal(got, gpu.from_numpy(np.ascontiguousarray(want, dtype=np.float32)).to(got.dtype))
    pages.close()


@pytest.mark.parametrize("dim", [64, 128])
def test_strides_runs_and_slots_out_of_range(gpu, dim):
    kv, n, page = 3, 75, 32
    pages = KVPages(1, 4, page, kv, dim)
    packed, x = to_type(gpu, kv_rows(3, n, 2 + 2 * kv, dim), "float32")
    k, v = packed[:, 2:2 + kv], packed[:, 2 + kv:]
    slots = np.arange(n) + 13  # runs over pages, not from a group's start
    slots[[4, 40, 74]] = [-1, 4 * page, 2**31 - 1]
    pages.append(0, i32(gpu, slots), k, v, stream=gpu.cuda.current_stream())
    gk, gv = _gathered(gpu, pages, 0, slots, "float32")
    good = (slots >= 0) & (slots < 4 * page)
    for got, want in ((gk, x[:, 2:2 + kv]), (gv, x[:, 2 + kv:])):
        ref = oracle.dequantize_q4_0(oracle.quantize_q4_0(want.astype(np.float32).reshape(-1))).reshape(want.shape)
        assert np.array_equal(got.numpy()[good], ref[good])
        assert not got.numpy()[~good].any()
    rest = np.setdiff1d(np.arange(4 * page), slots)
    assert not _gathered(gpu, pages, 0, rest)[0].numpy().any()
    # into strided rows, what lies between them left alone
    out = gpu.full((n, 2 + 2 * kv, dim), 7.0, device="cuda")
    pages.gather(0, i32(gpu, slots), out[:, 2:2 + kv], out[:, 2 + kv:], stream=gpu.cuda.current_stream())
    assert np.array_equal(out[:, 2:2 + kv].cpu().numpy(), gk.numpy()) and bool((out[:, :2] == 7.0).all())
    pages.close()


def test_odd_values_and_blocks_as_they_are(gpu):
    kv, dim, page = 2, 128, 16
    x = kv_rows(5, 6, kv, dim)
    x[0] = 0.0
    x[1, 0, :32] = np.nan
    x[2, 1, 5] = np.inf
    x[3] *= 1e-39
    x[4] *= 1e30
    pages = KVPages(1, 2, page, kv, dim)
    slots = np.array([3, 31, 0, 16, 8, 9])
    t = gpu.from_numpy(x).cuda()
    pages.append(0, i32(gpu, slots), t, t.flip(0).contiguous(), stream=gpu.cuda.current_stream())
    gk, gv = _gathered(gpu, pages, 0, slots)
    assert np.array_equal(gk.numpy(), _blocks(x)) and np.array_equal(gv.numpy(), _blocks(x[::-1]))
    # a ring's blocks move into the pages and come out the same
    ring = KVRing(1, 1, kv, dim, 40)
    r = kv_rows(6, 40, kv, dim)
    ring.write(0, 0, 0, gpu.from_numpy(r).cuda(), gpu.from_numpy(r).cuda(), stream=gpu.cuda.current_stream())
    gpu.cuda.synchronize()
    blocks = gpu.from_numpy(ring.export_q4_0(0, 0, 0, 8, 20)).cuda()
    more = KVPages(1, 3, page, kv, dim)
    at = i32(gpu, np.arange(20) + 5)
    more.append(0, at, blocks, blocks, stream=gpu.cuda.current_stream())
    back = gpu.zeros_like(blocks), gpu.zeros_like(blocks)
    more.gather(0, at, *back, stream=gpu.cuda.current_stream())
    assert gpu.equal(back[0], blocks) and gpu.equal(back[1], blocks)
    for p in (pages, more, ring):
        p.close()


def test_slots_past_32_bits_of_bytes(gpu):
    # 2^23 slots of 2 heads x 144 bytes a layer, and a second layer behind them
    pages = KVPages(2, 1 << 17, 128, 2, 128)
    assert pages.nbytes > 2**32
    slots = np.array([pages.n_pages * 128 - 1, pages.n_pages * 128 - 17, 1 << 24, 0, (1 << 23) + 5])
    x = kv_rows(8, len(slots), 2, 128)
    t = gpu.from_numpy(x).cuda()
    pages.append(1, i32(gpu, slots), t, t, stream=gpu.cuda.current_stream())
    good = slots < pages.n_pages * 128
    for got in _gathered(gpu, pages, 1, slots):
        assert np.array_equal(got.numpy()[good], _blocks(x)[good])
    assert not _gathered(gpu, pages, 0, slots[good])[0].numpy().any()
    pages.close()


def test_refusals(gpu):
    pages = KVPages(1, 2, 32, 2, 64)
    slots = i32(gpu, np.arange(4))
    rows = gpu.zeros(4, 2, 64, device="cuda")
    for layer in (-1, 1):
        with pytest.raises(RingError) as e:
            pages.append(layer, slots, rows, rows)
        assert e.value.rc == 2 and "layer" in e.value.msg
    with pytest.raises(RingError, match="aligned"):
        flat = gpu.zeros(4 * 2 * 64 + 1, device="cuda")[1:].view(4, 2, 64)
        pages.append(0, slots, flat, flat)
    for bad in (rows[:3], rows.double(), rows[:, :, ::2], gpu.zeros(4, 2, 128, device="cuda").transpose(0, 1)):
        with pytest.raises((ValueError, TypeError)):
            pages.append(0, slots, bad, bad)
    with pytest.raises(ValueError):
        pages.append(0, slots.long(), rows, rows)
    pages.append(0, slots[:0], rows[:0], rows[:0])  # nothing to do
    pages.close()

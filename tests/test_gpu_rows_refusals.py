"""Refusals of calls on handles: nothing is launched, and what was there stays."""
import pytest

import bmo_jetson_amd as bmo

pytestmark = pytest.mark.gpu


@pytest.fixture
def mem(gpu):
    """A megabyte that refused calls name."""
    t = gpu.full((1 << 20,), 7, dtype=gpu.uint8, device="cuda")
    yield t
    gpu.cuda.synchronize()
    assert bool((t == 7).all())


# (4 rows of 64 codes: 256 bytes, their scales 16; 128 outputs of 4 rows in fp32: 2048, of the gate 1024)
A, B, C, D, E = 0, 4096, 8192, 12288, 16384


@pytest.mark.parametrize("args,rc,why", [
    (dict(codes=None), 1, "null"), (dict(scales=None), 1, "null"), (dict(out=None), 1, "null"), (dict(n=-1), 2, "n_rows"),
    (dict(n=(1 << 20) + 1), 2, "n_rows"), (dict(type=3), 2, "fp32"), (dict(stride=127), 2, "shorter"),
    (dict(stride=(1 << 40) + 1), 2, "long"), (dict(codes=8), 2, "aligned"), (dict(scales=B + 1), 2, "aligned"),
    (dict(out=C + 2), 2, "aligned"), (dict(out=A), 2, "overlaps"), (dict(out=A + 252), 2, "overlaps"),
    (dict(out=B - 2044), 2, "overlaps"), (dict(stride=256, out=B), 2, "overlaps")])
def test_product(gpu, mem, args, rc, why):
    a = dict(n=4, codes=A, scales=B, type=0, out=C, stride=0)
    a.update(args)
    for k in ("codes", "scales", "out"):
        a[k] = None if a[k] is None else mem.data_ptr() + a[k]
    with bmo.Q4Weights(128, 64) as w:
        assert bmo.lib().bmo_weights_product(w.handle, *a.values(), None) == rc
        assert w.last_error().startswith("bmo_weights_product:") and why in w.last_error()


@pytest.mark.parametrize("args,rc,why", [
    (dict(out=None), 1, "null"), (dict(act=0), 2, "activation"), (dict(act=3), 2, "activation"),
    (dict(out_codes=D), 2, "together"), (dict(out_codes=D + 8, out_scales=E), 2, "aligned"), (dict(rows=96), 2, "whole blocks"),
    (dict(out_codes=A, out_scales=E), 2, "overlaps"), (dict(out_codes=D, out_scales=B), 2, "overlaps"),
    (dict(out_codes=C, out_scales=E), 2, "overlaps"), (dict(out_codes=D, out_scales=D + 254), 2, "overlaps"),
    (dict(out=None, out_codes=A + 240, out_scales=E), 2, "overlaps")])
def test_gated(gpu, mem, args, rc, why):
    a = dict(rows=128, n=4, codes=A, scales=B, act=1, type=0, out=C, stride=0, out_codes=None, out_scales=None)
    a.update(args)
    for k in ("codes", "scales", "out", "out_codes", "out_scales"):
        a[k] = None if a[k] is None else mem.data_ptr() + a[k]
    with bmo.Q4Weights(a.pop("rows"), 64) as w:
        assert bmo.lib().bmo_weights_gated(w.handle, *a.values(), None) == rc
        assert w.last_error().startswith("bmo_weights_gated:") and why in w.last_error()


@pytest.mark.parametrize("args,rc,why", [
    ((0, 1, None), 1, "null"), ((-1, 1, A), 2, "out of range"), ((0, -1, A), 2, "out of range"), ((100, 29, A), 2, "out of range"),
    ((2**31 - 1, 1, A), 2, "out of range"), ((0, 1, A + 1), 2, "aligned")])
def test_load(gpu, mem, args, rc, why):
    row, n, at = args
    with bmo.Q4Weights(128, 64) as w:
        assert bmo.lib().bmo_weights_load(w.handle, row, n, None if at is None else mem.data_ptr() + at, None) == rc
        assert w.last_error().startswith("bmo_weights_load:") and why in w.last_error()


# (4 tokens of 2 heads of 16 in fp32: 512 bytes; of 1 head 256)
@pytest.mark.parametrize("args,rc,why", [
    (dict(pos=None), 1, "null"), (dict(q=None), 1, "null"), (dict(qo=None), 1, "null"), (dict(k=None), 1, "null"),
    (dict(n=-1), 2, "n_tok"), (dict(heads=0), 2, "n_heads"), (dict(heads=4097), 2, "n_heads"), (dict(kv=-1), 2, "n_kv_heads"),
    (dict(n=1 << 30), 2, "too large"), (dict(type=5), 2, "fp32"), (dict(qs=31), 2, "shorter"), (dict(kos=15), 2, "shorter"),
    (dict(q=A + 2), 2, "aligned"), (dict(qo=A, qos=64), 2, "stride"), (dict(qo=A + 508), 2, "overlaps"),
    (dict(qo=B), 2, "overlaps"), (dict(ko=A), 2, "overlaps"), (dict(ko=A + 64), 2, "overlaps"), (dict(ko=C + 12), 2, "overlaps")])
def test_rope(gpu, mem, args, rc, why):
    a = dict(n=4, pos=C, type=0, heads=2, q=A, qs=0, qo=A, qos=0, kv=1, k=B, ks=0, ko=B, kos=0)
    a.update(args)
    for k in ("pos", "q", "qo", "k", "ko"):
        a[k] = None if a[k] is None else mem.data_ptr() + a[k]
    with bmo.Rope(16) as rope:
        assert bmo.lib().bmo_rope_apply(rope.handle, *a.values(), None) == rc
        assert rope.last_error().startswith("bmo_rope_apply:") and why in rope.last_error()


def test_packed_views_are_no_overlap(gpu):
    """q and k in one packed tensor, turned into another and in place."""
    torch = gpu
    torch.manual_seed(3)
    packed = torch.randn(5, 4, 16, device="cuda")
    other = packed.clone()
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    with bmo.Rope(16) as rope:
        result = torch.empty_like(packed)
        rope.apply(pos, packed[:, :2], packed[:, 2:3], result[:, :2], result[:, 2:3], stream=torch.cuda.current_stream())
        rope.apply(pos, other[:, :2], other[:, 2:3], stream=torch.cuda.current_stream())
        # into rows beside them
        rope.apply(pos, packed[:, :1], None, packed[:, 3:], stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
    assert torch.equal(other[:, :3], result[:, :3]) and torch.equal(packed[:, 3], result[:, 0])


@pytest.mark.parametrize("dim", [64, 61])
def test_x_as_its_own_residual(gpu, dim):
    """h = 2 x is exact, and so is the norm of a row of equal magnitudes: h^2 = 2.25, 1.5 / 1.5."""
    torch = gpu
    x = torch.full((3, dim), 0.75, device="cuda")
    x[:, ::2] = -0.75
    sign, out = x.sign(), torch.empty_like(x)
    bmo.rms_norm(x, torch.ones(dim, device="cuda"), eps=0.0, residual=x, out=out, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(x, 1.5 * sign)
    # (the sum of squares is exact; its division, root and reciprocal round three times, the product once)
    assert float((out - sign).abs().max()) <= 4 * 2.0**-24

"""The operators on rows without a GPU: refusals of the C ABI and of the
Python view, and that they come before anything is launched."""
import ctypes

import numpy as np
import pytest

import bmo_jetson_amd as bmo
from bmo_jetson_amd import rows

A = 0x10000  # an address that is never followed: every call here is refused
TOO_LONG = (1 << 40) + 1


def _norm(**k):
    a = dict(n=2, dim=64, type=0, x=A, xs=0, rt=0, res=None, rs=0, wt=0, w=A, eps=1e-5, ot=0, out=A, os=0, codes=None,
             scales=None)
    a.update(k)
    return bmo.lib().bmo_rms_norm(*a.values(), None)


@pytest.mark.parametrize("args,rc,why", [
    (dict(x=None), 1, "null"), (dict(w=None), 1, "null"), (dict(out=None), 1, "null"), (dict(codes=A), 2, "together"),
    (dict(n=-1), 2, "n_rows"), (dict(n=1 << 22), 2, "n_rows"), (dict(dim=0), 2, "dim"), (dict(dim=32769), 2, "dim"),
    (dict(dim=48, codes=A, scales=A), 2, "multiple of 32"), (dict(eps=-1.0), 2, "eps"), (dict(eps=float("nan")), 2, "eps"),
    (dict(type=3), 2, "fp32"), (dict(wt=9), 2, "fp32"), (dict(ot=-1), 2, "fp32"), (dict(res=A, rt=4), 2, "fp32"),
    (dict(xs=63), 2, "shorter"), (dict(res=A, rs=1), 2, "shorter"), (dict(os=TOO_LONG), 2, "long"),
    (dict(x=A + 2), 2, "aligned"), (dict(type=1, x=A + 1), 2, "aligned"), (dict(codes=A + 8, scales=A), 2, "aligned"),
    (dict(codes=A, scales=A + 1), 2, "aligned")])
def test_norm_refuses(args, rc, why):
    assert _norm(**args) == rc
    err = bmo.lib().bmo_rows_last_error().decode()
    assert err.startswith("bmo_rms_norm:") and why in err


# (2 rows of 64: 512 bytes of fp32, 128 of codes, 8 of scales)
B, C, D = A + 4096, A + 8192, A + 12288


@pytest.mark.parametrize("args", [
    dict(x=A, out=A + 256, w=B), dict(x=A, out=A, ot=1, w=B), dict(x=A, out=A, xs=128, w=B), dict(x=A, out=B, w=B + 508),
    dict(x=A, res=B, out=B, w=C), dict(x=A, res=A + 4, out=B, w=C), dict(x=A, res=A, rt=1, out=B, w=C),
    dict(x=A, res=B, out=C, w=B + 4), dict(x=A, out=None, codes=A + 496, scales=B, w=C),
    dict(x=A, out=None, codes=B, scales=A + 510, w=C), dict(x=A, out=C, codes=B, scales=B + 126, w=D),
    dict(x=A, out=B, codes=B + 496, scales=C, w=D)])
def test_norm_refuses_overlaps(args):
    assert _norm(**args) == 2
    assert "overlaps" in bmo.lib().bmo_rows_last_error().decode()


@pytest.mark.parametrize("x,codes,scales", [(A, A, B), (A, A + 496, B), (A, B, A + 510), (A, B, B + 126), (A + 64, A, B)])
def test_quantize_refuses_overlaps(x, codes, scales):
    assert bmo.lib().bmo_quantize_rows(2, 64, 0, x, 0, codes, scales, None) == 2
    assert "overlaps" in bmo.lib().bmo_rows_last_error().decode()


@pytest.mark.parametrize("args,rc,why", [
    ((2, 64, 0, None, 0, A, A), 1, "null"), ((2, 64, 0, A, 0, None, A), 1, "null"), ((2, 64, 0, A, 0, A, None), 1, "null"),
    ((-1, 64, 0, A, 0, A, A), 2, "n_rows"), ((2, 48, 0, A, 0, A, A), 2, "multiple"), ((2, 0, 0, A, 0, A, A), 2, "multiple"),
    ((2, 64, 3, A, 0, A, A), 2, "fp32"), ((2, 64, 0, A, 32, A, A), 2, "shorter"), ((2, 64, 0, A, 0, A + 1, A), 2, "aligned"),
    ((1 << 20, 1 << 14, 0, A, 0, A, A), 2, "too large")])
def test_quantize_refuses(args, rc, why):
    assert bmo.lib().bmo_quantize_rows(*args, None) == rc
    err = bmo.lib().bmo_rows_last_error().decode()
    assert err.startswith("bmo_quantize_rows:") and why in err


@pytest.mark.parametrize("args,why", [
    ((0, 64, 1, 1e4, 1.0, 0, 0, 0, 0), "head_dim"), ((1026, 64, 1, 1e4, 1.0, 0, 0, 0, 0), "head_dim"),
    ((64, 65, 1, 1e4, 1.0, 0, 0, 0, 0), "rot_dim"), ((64, 33, 1, 1e4, 1.0, 0, 0, 0, 0), "rot_dim"),
    ((64, 0, 1, 1e4, 1.0, 0, 0, 0, 0), "rot_dim"), ((64, 64, 1, 1.0, 1.0, 0, 0, 0, 0), "theta"),
    ((64, 64, 1, float("inf"), 1.0, 0, 0, 0, 0), "theta"), ((64, 64, 1, 1e4, 0.0, 0, 0, 0, 0), "factor"),
    ((64, 64, 1, 1e4, float("nan"), 0, 0, 0, 0), "factor"), ((64, 64, 1, 1e4, 2.0, -1, 0, 0, 0), "trained"),
    ((64, 64, 1, 1e4, 0.5, 0, 0, 0, 0), "radian"), ((64, 64, 1, 1e4, 2.0, 4096, 0, 0, 1e39), "magnitude")])
def test_rope_create_refuses(args, why):
    L = bmo.lib()
    assert not L.bmo_rope_create(*args, None)
    err = L.bmo_rope_last_error(None).decode()
    assert err.startswith("bmo_rope_create:") and why in err


@pytest.mark.parametrize("divisor", [0.0, 0.5, -1.0, float("nan")])
def test_rope_divisors_refused(divisor):
    with pytest.raises(RuntimeError, match="radian"):
        bmo.Rope(4, divisors=[divisor, 1.0])
    with pytest.raises(ValueError, match="2 numbers"):
        bmo.Rope(4, divisors=[1.0])


@pytest.mark.parametrize("args,why", [((0, 64), "rows"), (((1 << 24) + 1, 64), "rows"), ((4, 0), "cols"), ((4, 33), "cols"),
                                      ((4, (1 << 24) + 32), "cols")])
def test_weights_create_refuses(args, why):
    L = bmo.lib()
    assert not L.bmo_weights_create(*args)
    err = L.bmo_weights_last_error(None).decode()
    assert err.startswith("bmo_weights_create:") and why in err
    with pytest.raises(RuntimeError, match="bmo_weights_create failed"):
        bmo.Q4Weights(*args)


def test_null_handles():
    L = bmo.lib()
    L.bmo_rope_free(None)
    L.bmo_weights_free(None)
    assert L.bmo_rope_device(None) == -1 and L.bmo_weights_device(None) == -1 and L.bmo_weights_bytes(None) == 0
    assert L.bmo_rope_apply(None, 0, None, 0, 1, None, 0, None, 0, 0, None, 0, None, 0, None) == 1
    assert L.bmo_weights_load(None, 0, 0, None, None) == 1
    assert L.bmo_weights_product(None, 0, None, None, 0, None, 0, None) == 1
    assert L.bmo_weights_gated(None, 0, None, None, 1, 0, None, 0, None, None, None) == 1


def test_tensors_that_are_refused(monkeypatch):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(rows, "_current", lambda: -1)
    x, w = torch.zeros(3, 64), torch.zeros(64)
    codes, scales = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.float16)
    same = torch.zeros(1, 64).expand(3, 64)
    weights = bmo.Q4Weights.__new__(bmo.Q4Weights)
    weights._h, weights._device, weights.rows, weights.cols = None, -1, 128, 64
    rope = bmo.Rope.__new__(bmo.Rope)
    rope._h, rope._device, rope.head_dim = None, -1, 16
    pos, q = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 16)
    cases = [(lambda: bmo.rms_norm(x, w), "must be given"),
             (lambda: bmo.rms_norm(x, w[:32], out=x), "64 elements"),
             (lambda: bmo.rms_norm(x, w.double(), out=x), "float tensor"),
             (lambda: bmo.rms_norm(x, w, out=x[:2]), r"out must be \[3\]\[64\]"),
             (lambda: bmo.rms_norm(x, w, out=same), "overlap"),
             (lambda: bmo.rms_norm(x, w, residual=same, out=x), "overlap"),
             (lambda: bmo.rms_norm(x.t(), w, out=x), "contiguous"),
             (lambda: bmo.rms_norm(x, w, codes=codes), "together"),
             (lambda: bmo.rms_norm(x, w, codes=codes, scales=scales[:, :1]), "one for each 32"),
             (lambda: bmo.quantize_rows(x, codes[:2], scales[:2]), "codes must be"),
             (lambda: bmo.quantize_rows(x[:, ::2], codes[:, :32].contiguous(), scales[:, :1].contiguous()), "contiguous"),
             (lambda: bmo.quantize_rows(x, torch.zeros(3, 128, dtype=torch.int8)[:, ::2], scales), "contiguous"),
             (lambda: weights.load(torch.zeros(1, 2, 17, dtype=torch.uint8)), "blocks"),
             (lambda: weights.product(codes, scales, x), r"out must be \[3\]\[128\]"),
             (lambda: weights.product(codes[:, :32].contiguous(), scales[:, :1].contiguous(), x), "codes must be"),
             (lambda: weights.gated(codes, scales), "must be given"),
             (lambda: weights.gated(codes, scales, out=x, activation="relu"), "silu, gelu"),
             (lambda: weights.gated(codes, scales, codes, None), "together"),
             (lambda: rope.apply(pos.long(), q), "int32"),
             (lambda: rope.apply(pos, q[:2]), r"q must be \[3\]"),
             (lambda: rope.apply(pos, q[:, :, :8]), "q must be"),
             (lambda: rope.apply(pos, q, q_out=q[:, :2]), "q_out must be"),
             (lambda: rope.apply(pos, q[:1].expand(3, 4, 16)), "overlap"),
             (lambda: rope.apply(pos, q, q.half()), "one type")]
    for i, (call, why) in enumerate(cases):
        with pytest.raises(ValueError, match=why):
            call()
            raise AssertionError(f"case {i} was not refused")
    for call in (lambda: bmo.rms_norm(x.double(), w, out=x), lambda: bmo.quantize_rows(x, codes.byte(), scales),
                 lambda: bmo.quantize_rows(x, codes, scales.float())):
        with pytest.raises(TypeError):
            call()
    monkeypatch.setattr(rows, "_current", lambda: 0)  # tensors that are elsewhere
    weights._device = rope._device = 0
    for call in (lambda: bmo.rms_norm(x, w, out=x), lambda: bmo.quantize_rows(x, codes, scales), lambda: rope.apply(pos, q),
                 lambda: weights.product(codes, scales, x)):
        with pytest.raises(ValueError, match="device 0"):
            call()


def test_oracle_of_8_bit_rows():
    """The helper's own quantizer: known scales and codes."""
    from _rows import scale8, split8
    assert scale8(np.float32(127.0)) == 1.0 and scale8(np.float32(0.0)) == 0.0
    assert scale8(np.float32(127.0) * np.float32(1.0001)) == np.nextafter(np.float16(1), np.float16(2))
    assert scale8(np.float32(1e-30)) == np.float16(2.0**-24)
    assert scale8(np.float32(127 * 65504.0)) == 65504.0 and np.isnan(scale8(np.float32(8.4e6)))
    x = np.zeros((1, 32), np.float32)
    x[0, :5] = [127, -126.6, 0.4, 0.5, 1.5]
    q, d = split8(x)
    assert d[0, 0] == 1.0 and list(q[0, :5]) == [127, -127, 0, 0, 2]

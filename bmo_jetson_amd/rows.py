"""Python view of the operators on rows between two attentions (ctypes over
include/bmo_attn.h): RMS norm, 8-bit rows, rotary positions, and products with
Q4_0 weights, plain and gated.

8-bit rows are a pair of contiguous tensors, codes (int8 [rows][cols]) and
scales (float16 [rows][cols // 32]); what they stand for is
``codes.view(rows, -1, 32) * scales[..., None]``.

A layer of a server's step, for the rows x of its entries::

    rms_norm(x, w1, residual=h, codes=c, scales=s)        # x: the layer before's
    qkv.product(c, s, packed)                             # q, k, v: views of packed
    rope.apply(positions, q, k, q_out, k_out)
    pages.append_decode(...)  or  pages.append(...), pages.attend(...)
    quantize_rows(attended, c, s); out.product(c, s, x)
    rms_norm(x, w2, residual=h, codes=c, scales=s)
    gate_up.gated(c, s, codes, scales); down.product(codes, scales, x)
"""
from __future__ import annotations

import ctypes

from ._lib import lib
from .pages import _code
from .ring import RingError, _stream

_ACTIVATIONS = {"silu": 1, "gelu": 2}
_SMALL: dict = {}  # what is asked of torch: the dtype objects of codes and scales, the current device


def _small(name: str):
    known = _SMALL.get(name)
    if known is None:
        import torch
        known = _SMALL[name] = getattr(torch, name)
    return known


def _current() -> int:
    """The current device."""
    known = _SMALL.get("device")
    if known is None:
        import torch
        known = _SMALL["device"] = torch.cuda.current_device
    return known()


def _shape(what: str, shape, n, cols) -> ValueError:
    want = f"[{'rows' if n is None else n}][{'columns' if cols is None else cols}]"
    return ValueError(f"{what} must be {want}, got {tuple(shape)}")


def _on(x, device: int, what: str) -> ValueError:
    return ValueError(f"{what} must be on device {device}, not on {x.device}")


# (The checks below cost as much as the launch of a short kernel: each asks a
# tensor as little as it can.)

def _rows(x, device: int, what: str, n=None, cols=None):
    """(address, stride, type, rows, columns) of a 2-d tensor of values."""
    shape = x.shape
    if len(shape) != 2:
        raise _shape(what, shape, n, cols)
    rows, width = shape
    if (n is not None and rows != n) or (cols is not None and width != cols):
        raise _shape(what, shape, n, cols)
    type_ = _code(x)
    if type_ > 2:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    stride = 0
    if not x.is_contiguous():
        stride, inner = x.stride()
        if width > 1 and inner != 1:
            raise ValueError(f"{what}: a row's elements must be contiguous")
        if rows > 1 and stride < width:
            raise ValueError(f"{what}: rows must not overlap (an expanded tensor)")
        if rows == 1:
            stride = 0
    if x.get_device() != device:
        raise _on(x, device, what)
    return x.data_ptr(), stride, type_, rows, width


def _rows8(codes, scales, device: int, what: str, n=None, cols=None):
    """(codes, scales, rows, columns) of 8-bit rows: addresses and sizes."""
    shape = codes.shape
    if len(shape) != 2:
        raise _shape(f"{what}: codes", shape, n, cols)
    rows, width = shape
    if (n is not None and rows != n) or (cols is not None and width != cols):
        raise _shape(f"{what}: codes", shape, n, cols)
    if scales.shape != (rows, width // 32) or width % 32:
        raise ValueError(f"{what}: scales must be one for each 32 codes of a row, got {tuple(scales.shape)}")
    if codes.dtype is not _small("int8") or scales.dtype is not _small("float16"):
        raise TypeError(f"{what} must be int8 and float16, got {codes.dtype} and {scales.dtype}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise ValueError(f"{what}: codes and scales must be contiguous")
    if codes.get_device() != device:
        raise _on(codes, device, what)
    if scales.get_device() != device:
        raise _on(scales, device, what)
    return codes.data_ptr(), scales.data_ptr(), rows, width


def _check(fn: str, rc: int) -> None:
    if rc != 0:
        e = lib().bmo_rows_last_error()
        raise RingError(fn, rc, e.decode() if e else None)


def rms_norm(x, weight, eps: float = 1e-5, residual=None, out=None, codes=None, scales=None, stream=None) -> None:
    """RMS norm of rows x [n][dim] on the current device.  residual [n][dim]
    (any of the three types) gets x added and is what is normalized, without it
    x is; the result, times weight [dim], goes to out [n][dim] (which may be x),
    to the 8-bit rows (codes, scales), or to both."""
    device = _current()
    xp, x_stride, x_type, n, dim = _rows(x, device, "x")
    rp, r_stride, r_type, _, _ = _rows(residual, device, "residual", n, dim) if residual is not None else (None, 0, 0, 0, 0)
    op, o_stride, o_type, _, _ = _rows(out, device, "out", n, dim) if out is not None else (None, 0, 0, 0, 0)
    if weight.shape != (dim,) or not weight.is_contiguous() or _code(weight) > 2:
        raise ValueError(f"weight must be a contiguous float tensor of {dim} elements")
    if weight.get_device() != device:
        raise _on(weight, device, "weight")
    if (codes is None) != (scales is None):
        raise ValueError("codes and scales come together")
    if out is None and codes is None:
        raise ValueError("out, or codes and scales, must be given")
    cp, sp = _rows8(codes, scales, device, "8-bit rows", n, dim)[:2] if codes is not None else (None, None)
    _check("bmo_rms_norm", lib().bmo_rms_norm(n, dim, x_type, xp, x_stride, r_type, rp, r_stride, _code(weight),
                                              weight.data_ptr(), float(eps), o_type, op, o_stride, cp, sp, _stream(stream)))


def quantize_rows(x, codes, scales, stream=None) -> None:
    """Rows x [n][cols] (cols a multiple of 32) as 8-bit rows, on the current device."""
    device = _current()
    xp, stride, type_, n, cols = _rows(x, device, "x")
    cp, sp, _, _ = _rows8(codes, scales, device, "8-bit rows", n, cols)
    _check("bmo_quantize_rows", lib().bmo_quantize_rows(n, cols, type_, xp, stride, cp, sp, _stream(stream)))


class _Handle:
    """What holds a C handle; subclasses name its calls."""

    _NAME = ""

    def _take(self, h) -> None:
        L = lib()
        if not h:
            err = getattr(L, self._NAME + "_last_error")(None)
            raise RuntimeError(f"{self._NAME}_create failed: {err.decode() if err else 'unknown'}")
        self._h = h
        self._free = getattr(L, self._NAME + "_free")  # (__del__ needs no module globals)
        self._device = getattr(L, self._NAME + "_device")(h)

    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            self._h = None
            self._free(h)

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter teardown: nothing left to report to
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self) -> int:
        return self._h

    def last_error(self) -> str | None:
        e = getattr(lib(), self._NAME + "_last_error")(self._h)
        return e.decode() if e else None

    def _check(self, call: str, rc: int) -> None:
        if rc != 0:
            raise RingError(call, rc, self.last_error())


class Rope(_Handle):
    """Rotary positions of heads of head_dim elements, the first rot_dim (all,
    if None) of which turn: neighbours (2i, 2i + 1) if interleaved, else (i, i +
    rot_dim / 2).  For long contexts the rates are divided by factor, or with
    trained (the length that the model was trained at) blended as YaRN does;
    divisors (a sequence of rot_dim / 2 numbers) divides them pair by pair."""

    _NAME = "bmo_rope"

    def __init__(self, head_dim: int, rot_dim: int | None = None, theta: float = 10000.0, interleaved: bool = True,
                 factor: float = 1.0, trained: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 magnitude: float = 0.0, divisors=None):
        rot_dim = head_dim if rot_dim is None else rot_dim
        table = None
        if divisors is not None:
            values = [float(x) for x in divisors]
            if len(values) != rot_dim // 2:
                raise ValueError(f"divisors must be {rot_dim // 2} numbers")
            table = (ctypes.c_double * len(values))(*values)
        self._take(lib().bmo_rope_create(head_dim, rot_dim, int(bool(interleaved)), float(theta), float(factor),
                                         int(trained), float(beta_fast), float(beta_slow), float(magnitude), table))
        self.head_dim, self.rot_dim = head_dim, rot_dim

    def _heads(self, x, n: int, what: str, like=None):
        """(address, stride, type, heads) of rows [tokens][heads][head_dim]."""
        shape = x.shape
        if len(shape) != 3 or shape[0] != n or shape[2] != self.head_dim or (like is not None and shape != like.shape):
            raise ValueError(f"{what} must be [{n}][{'heads' if like is None else like.shape[1]}][{self.head_dim}], "
                             f"got {tuple(shape)}")
        heads, stride = shape[1], 0
        if not x.is_contiguous():
            stride, per_head, inner = x.stride()
            if n and (inner != 1 or (heads > 1 and per_head != self.head_dim)):
                raise ValueError(f"{what}: a token's heads must be contiguous")
            if n > 1 and stride < heads * self.head_dim:
                raise ValueError(f"{what}: rows must not overlap (an expanded tensor)")
            if n <= 1:
                stride = 0
        type_ = _code(x)
        if type_ > 2:
            raise TypeError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
        if x.get_device() != self._device:
            raise _on(x, self._device, what)
        return x.data_ptr(), stride, type_, heads

    def apply(self, positions, q, k=None, q_out=None, k_out=None, stream=None) -> None:
        """Turns q [n_tok][heads][head_dim], and k, by positions [n_tok] (int32),
        in place or into q_out and k_out."""
        n = positions.numel()
        if _code(positions) != 4 or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 tensor")
        if positions.get_device() != self._device:
            raise _on(positions, self._device, "positions")
        qp, q_stride, type_, heads = self._heads(q, n, "q")
        if k is None and k_out is not None:
            raise ValueError("k_out without k")
        parts = [(qp, q_stride) if q_out is None else self._heads(q_out, n, "q_out", q)]
        kp, k_stride, k_type, k_heads = (None, 0, type_, 0) if k is None else self._heads(k, n, "k")
        parts.append((kp, k_stride) if k is None or k_out is None else self._heads(k_out, n, "k_out", k))
        if k_type != type_ or any(len(p) > 2 and p[2] != type_ for p in parts):
            raise ValueError("q, k and what they go to must have one type")
        self._check("bmo_rope_apply", lib().bmo_rope_apply(
            self._h, n, positions.data_ptr(), type_, heads, qp, q_stride, parts[0][0], parts[0][1], k_heads, kp, k_stride,
            parts[1][0], parts[1][1], _stream(stream)))


class Q4Weights(_Handle):
    """A Q4_0 weight matrix [rows][cols] on the current device, for 8-bit rows
    of any number.  For a gated feed-forward the first half of the rows are the
    gate's, the second half those of what it lets through."""

    _NAME = "bmo_weights"

    def __init__(self, rows: int, cols: int):
        self._take(lib().bmo_weights_create(rows, cols))
        self.rows, self.cols = rows, cols

    @property
    def nbytes(self) -> int:
        return int(lib().bmo_weights_bytes(self._h))

    def load(self, blocks, row: int = 0, stream=None) -> None:
        """Rows from `row` on from ggml blocks, uint8 [n][cols // 32][18]."""
        shape = (blocks.shape[0], self.cols // 32, 18)
        if tuple(blocks.shape) != shape or _code(blocks) != 3 or not blocks.is_contiguous():
            raise ValueError(f"blocks must be a contiguous uint8 tensor {shape}")
        if blocks.get_device() != self._device:
            raise _on(blocks, self._device, "blocks")
        self._check("bmo_weights_load", lib().bmo_weights_load(self._h, int(row), shape[0], blocks.data_ptr(),
                                                               _stream(stream)))

    def product(self, codes, scales, out, stream=None) -> None:
        """out [n][rows] = the 8-bit rows times the matrix."""
        cp, sp, n, _ = _rows8(codes, scales, self._device, "8-bit rows", None, self.cols)
        op, stride, type_, _, _ = _rows(out, self._device, "out", n, self.rows)
        self._check("bmo_weights_product", lib().bmo_weights_product(self._h, n, cp, sp, type_, op, stride,
                                                                     _stream(stream)))

    def gated(self, codes, scales, out_codes=None, out_scales=None, out=None, activation: str = "silu",
              stream=None) -> None:
        """act(gate) * up, [n][rows // 2], into 8-bit rows for the projection
        down (out_codes, out_scales), into out, or both."""
        act = _ACTIVATIONS.get(activation)
        if act is None:
            raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}")
        if (out_codes is None) != (out_scales is None):
            raise ValueError("out_codes and out_scales come together")
        if out is None and out_codes is None:
            raise ValueError("out, or out_codes and out_scales, must be given")
        cp, sp, n, _ = _rows8(codes, scales, self._device, "8-bit rows", None, self.cols)
        half = self.rows // 2
        op, stride, type_ = _rows(out, self._device, "out", n, half)[:3] if out is not None else (None, 0, 0)
        ocp, osp = (None, None) if out_codes is None else _rows8(out_codes, out_scales, self._device, "output rows", n,
                                                                 half)[:2]
        self._check("bmo_weights_gated", lib().bmo_weights_gated(self._h, n, cp, sp, act, type_, op, stride, ocp, osp,
                                                                 _stream(stream)))

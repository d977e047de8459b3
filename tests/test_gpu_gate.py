"""The gate's activation alone, relative to its own value: products that are
exact, so that what is left is the activation's arithmetic."""
import numpy as np
import pytest

from _rows import U, blocks_of, check
from _shapes import product_shapes
from test_gpu_weights import GATED_SHAPES, _weights

pytestmark = pytest.mark.gpu

KERNELS = [(1, 1056, 416, None)] + list({c[3]: c for c in reversed(GATED_SHAPES)}.values())


@pytest.mark.parametrize("n,hidden,cols,shape", KERNELS)
def test_silu_keeps_its_bits(gpu, n, hidden, cols, shape):
    torch = gpu
    assert shape is None or product_shapes([(True, n, hidden, cols)]) == [shape]
    r = np.random.default_rng(n)
    # one weight of a row that is not zero: a gate is (code - 8) * q * d8, 4 + 7 + 11 bits
    wc = np.full((2 * hidden, cols // 32, 32), 8, np.uint8)
    at = r.integers(0, cols, 2 * hidden)
    w = np.concatenate((r.choice([-8, -7, -5, -3, -1, 1, 2, 5, 7], hidden), r.choice([-8, -3, 1, 7], hidden)))
    w[:2] = -8, 7  # the ends of the range
    wc.reshape(2 * hidden, cols)[np.arange(2 * hidden), at] = w + 8
    handle = _weights(torch, blocks_of(wc, np.ones((2 * hidden, cols // 32), np.float16)))
    codes = r.integers(1, 128, (n, cols)).astype(np.int8)
    scales = (86.9 / (8 * 127) * r.uniform(0.25, 1, (n, cols // 32))).astype(np.float16)
    codes[:, at[:2]], scales[:, at[:2] // 32] = 127, 86.9 / (8 * 127)
    out = torch.empty(n, hidden, device="cuda")
    handle.gated(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), out=out,
                 stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    values = (codes.reshape(n, -1, 32) * scales.astype(np.float64)[:, :, None]).reshape(n, cols)
    both = values[:, at] * w
    g, u = both[:, :hidden], both[:, hidden:]
    assert -87 <= g.min() < -86 and g.max() > 76
    h = g / (1 + np.exp(-g)) * u
    # e^-g: the hardware's 2^x 2 U, its factor and their product U each; the divisor U, the reciprocal 2 U, two products
    # U each; and a U for what their products leave out
    check(out.double().cpu().numpy(), h, 10 * U * np.abs(h), f"{n} {hidden} {cols}")


def test_ends_of_the_range(gpu):
    """Past exp's overflow nothing is let through, past its underflow everything; infinities and NaN as the formula has them."""
    torch = gpu
    wc = np.full((64, 1, 32), 8, np.uint8)
    wc[:, 0, 0], wc[32:, 0, 0], wc[32:, 0, 1] = 9, 8, 9  # gate: element 0, what it lets through: element 1
    wc[16:32, 0, 0] = 7
    w = _weights(torch, blocks_of(wc, np.ones((64, 1), np.float16)))
    codes = np.zeros((6, 32), np.int8)
    codes[:, :2] = [[88, 1], [89, 1], [110, 1], [127, 1], [127, 1], [0, 1]]
    scales = np.ones((6, 1), np.float16)
    scales[4] = 65504.0
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    for activation in ("silu", "gelu"):
        for n in (1, 6):
            out = torch.empty(n, 32, device="cuda")
            for i in range(6 // n):
                w.gated(c[i:i + n], s[i:i + n], out=out, activation=activation, stream=torch.cuda.current_stream())
                torch.cuda.synchronize()
                got, rows = out.cpu().numpy(), np.arange(i, i + n)
                full = (codes[rows, 0] * scales[rows, 0].astype(np.float32) * scales[rows, 0].astype(np.float32))[:, None]
                assert (np.abs(got[:, :16] - full) <= 4 * U * full).all()
                # 88 e^-88 = 5e-37
                assert (np.abs(got[:, 16:]) <= 1e-36).all() and (got[rows > 0, 16:] == 0).all()

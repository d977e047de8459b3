"""Every kernel of a product, plain and gated, at its edges: columns that end
anywhere in a unit, codes and scales at the ends of their ranges, scales that
are NaN or infinite, calls at once and captured."""
import numpy as np
import pytest

from _rows import blocks_of, check, check8, gated, product, q4_0, rounded
from _shapes import product_shapes
from test_gpu_weights import GATED_SHAPES, SHAPES, _product, _rows8, _weights

pytestmark = pytest.mark.gpu

# Units of 128 columns that are whole or half full, beside the quarters of SHAPES (rows, outputs, columns, kernel).
HALVES = [(2, 48, 128, (16, 16, 8)), (5, 48, 64, (16, 16, 8)), (2, 4097, 128, (16, 32, 8)), (2, 4097, 64, (16, 32, 8)),
          (2, 8193, 1152, (16, 64, 8)), (2, 8193, 1088, (16, 64, 8)), (17, 4097, 128, (32, 32, 4)), (17, 4097, 64, (32, 32, 4)),
          (17, 4097, 640, (32, 32, 8)), (17, 4097, 576, (32, 32, 8)), (65, 8193, 512, (32, 64, 4)), (65, 8193, 448, (32, 64, 4)),
          (2, 8193, 128, (32, 128, 1)), (2, 8193, 64, (32, 128, 1)), (97, 8193, 128, (32, 256, 1)), (97, 8193, 64, (32, 256, 1)),
          (1501, 2049, 4096, (64, 128, 2)), (1501, 2049, 4032, (64, 128, 2)), (1501, 4097, 128, (64, 256, 1)),
          (1501, 4097, 64, (64, 256, 1))]
GATED_HALVES = [(2, 32, 128, (16, 32, 8)), (2, 32, 64, (16, 32, 8)), (17, 4128, 128, (32, 32, 4)), (17, 4128, 64, (32, 32, 4)),
                (17, 4128, 640, (32, 32, 8)), (17, 4128, 576, (32, 32, 8)), (65, 6016, 128, (32, 64, 2)),
                (65, 6016, 64, (32, 64, 2)), (325, 3104, 128, (32, 128, 1)), (325, 3104, 64, (32, 128, 1)),
                (197, 6016, 2176, (64, 64, 2)), (197, 6016, 2112, (64, 64, 2)), (515, 6016, 256, (64, 128, 1)),
                (515, 6016, 192, (64, 128, 1))]
# One row: 8 waves to a tile, 16, and a row too long for that kernel.
ONE = [(1, 97, 320, None), (1, 97, 4160, None), (1, 48, 32864, None)]
GATED_ONE = [(1, 1056, 416, None), (1, 96, 4160, None), (1, 32, 32864, None)]
# Of each kernel a case that ends in a quarter of a unit.
QUARTERS = list({c[3]: c for c in reversed(SHAPES)}.values())
GATED_QUARTERS = list({c[3]: c for c in reversed(GATED_SHAPES)}.values())


def _takes(shape, is_gated, n, outs, cols):
    assert shape is None or product_shapes([(is_gated, n, outs, cols)]) == [shape]


@pytest.mark.parametrize("n,rows,cols,shape", HALVES)
def test_columns(gpu, n, rows, cols, shape):
    _takes(shape, False, n, rows, cols)
    _product(gpu, n, rows, cols, seed=n)


@pytest.mark.parametrize("n,hidden,cols,shape", GATED_HALVES)
def test_gated_columns(gpu, n, hidden, cols, shape):
    torch = gpu
    _takes(shape, True, n, hidden, cols)
    blocks, wc, ws = q4_0(n, 2 * hidden, cols)
    w = _weights(torch, blocks)
    codes, scales, c, s = _rows8(torch, n + 1, n, cols)
    both, off = product(codes, scales, wc, ws)
    h, bound = gated(both[:, :hidden], both[:, hidden:], off[:, :hidden], off[:, hidden:], "silu")
    out = torch.empty(n, hidden, device="cuda")
    oc = torch.empty(n, hidden, dtype=torch.int8, device="cuda")
    os = torch.empty(n, hidden // 32, dtype=torch.float16, device="cuda")
    w.gated(c, s, oc, os, out=out, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    check(out.double().cpu().numpy(), h, rounded(bound, h, "float32"), "out")
    check8(oc.cpu().numpy(), os.cpu().numpy(), h, bound, "8-bit rows")


def _extreme(n, rows, cols):
    """Weights and 8-bit rows at the ends of their ranges, signs mixed."""
    r = np.random.default_rng(n + cols)
    wc = r.choice([0, 15, 8], (rows, cols // 32, 32)).astype(np.uint8)
    wc[3], wc[4] = 0, 15
    ws = r.choice([65504.0, -65504.0, 2.0**-24, 1.0, 0.0, -0.0], (rows, cols // 32)).astype(np.float16)
    codes = r.choice([-127, 127, -128, 0, 1], (n, cols)).astype(np.int8)
    codes[0] = 127
    scales = r.choice([65504.0, 2.0**-24, 0.5, 0.0], (n, cols // 32)).astype(np.float16)
    return r, wc, ws, codes, scales


def _out(torch, w, codes, scales):
    out = torch.empty(codes.shape[0], w.rows, device="cuda")
    w.product(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), out, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return out.double().cpu().numpy()


@pytest.mark.parametrize("n,rows,cols,shape", ONE + HALVES + QUARTERS)
def test_extreme_codes_and_scales(gpu, n, rows, cols, shape):
    _takes(shape, False, n, rows, cols)
    _, wc, ws, codes, scales = _extreme(n, rows, cols)
    w = _weights(gpu, blocks_of(wc, ws))
    for lowest in (False, True) if n == 1 else (False,):
        if lowest:
            codes[0] = -128
        ref, bound = product(codes, scales, wc, ws)
        assert np.isfinite(ref).all()
        check(_out(gpu, w, codes, scales), ref, bound, "extreme")


@pytest.mark.parametrize("n,rows,cols,shape", ONE + HALVES + QUARTERS)
def test_scales_that_are_not_finite(gpu, n, rows, cols, shape):
    """Of the rows by IEEE rules (an infinite scale makes infinities, or NaN
    where a block's sum or its other scale is zero), of the weights always NaN;
    rows and columns beside them keep their values."""
    _takes(shape, False, n, rows, cols)
    r, wc, ws, codes, scales = _extreme(n, rows, cols)
    last = cols // 32 - 1
    ws[7, last], ws[9, 0], ws[12, last] = np.nan, np.inf, -np.inf
    w = _weights(gpu, blocks_of(wc, ws))
    for turn in range(4 if n == 1 else 1):
        scales8 = scales.copy()
        for i in range(n):
            kind = (i + turn) % 4
            if kind:
                scales8[i, {1: r.integers(0, last + 1), 2: last, 3: 0}[kind]] = np.nan if kind == 1 else np.inf
        with np.errstate(invalid="ignore"):
            ref, bound = product(codes, scales8, wc, ws)
        ref[:, [7, 9, 12]] = np.nan
        kinds = (np.arange(n) + turn) % 4
        assert np.isnan(ref[kinds == 1]).all() and np.isfinite(np.delete(ref[kinds == 0], [7, 9, 12], axis=1)).all()
        assert not np.isfinite(ref[kinds > 1]).any()
        assert n < 4 or (np.isinf(ref).any() and np.isnan(np.delete(ref, [7, 9, 12], axis=1)[kinds > 1]).any())
        check(_out(gpu, w, codes, scales8), ref, np.nan_to_num(bound, nan=0.0, posinf=0.0), "not finite")


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("n,hidden,cols,shape", GATED_ONE + GATED_HALVES + GATED_QUARTERS)
def test_gated_far_out(gpu, n, hidden, cols, shape, activation):
    """Gates so large that exp overflows, results past 8 bits' scales, zeros, scales that are not finite."""
    torch = gpu
    _takes(shape, True, n, hidden, cols)
    nb = cols // 32
    wc, ws = np.full((2 * hidden, nb, 32), 9, np.uint8), np.ones((2 * hidden, nb), np.float16)
    ws[1::2] = -1.0
    w = _weights(torch, blocks_of(wc, ws))
    codes = np.full((n, cols), 100, np.int8)
    for turn in range(6 if n < 6 else 1):
        kinds = (np.arange(n) + turn) % 6
        scales = np.ones((n, nb), np.float16)
        scales[kinds == 1], scales[kinds == 2], scales[kinds == 4] = 0.0, 60000.0, 2.0**-24
        scales[kinds == 3, 0], scales[kinds == 5, -1] = np.nan, np.inf
        both, off = product(codes, scales, wc, ws)
        with np.errstate(invalid="ignore"):
            h, bound = gated(both[:, :hidden], both[:, hidden:], off[:, :hidden], off[:, hidden:], activation)
        out = torch.empty(n, hidden, device="cuda")
        oc = torch.full((n, hidden), 77, dtype=torch.int8, device="cuda")
        os = torch.empty(n, hidden // 32, dtype=torch.float16, device="cuda")
        w.gated(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), oc, os, out=out, activation=activation,
                stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        check(out.double().cpu().numpy(), h, rounded(bound, h, "float32"), activation)
        check8(oc.cpu().numpy(), os.cpu().numpy(), h, bound, activation)


@pytest.mark.parametrize("n,rows,cols,shape", ONE + QUARTERS)
def test_calls_at_once_and_captured(gpu, n, rows, cols, shape):
    torch = gpu
    _takes(shape, False, n, rows, cols)
    w = _weights(torch, q4_0(n, rows, cols)[0])
    ins = [_rows8(torch, n + i, n, cols)[2:] for i in range(2)]
    _at_once_and_captured(torch, lambda i, outs: w.product(*ins[i], outs[0], stream=torch.cuda.current_stream()),
                          lambda: (torch.zeros(n, rows, device="cuda"),))


@pytest.mark.parametrize("n,hidden,cols,shape", GATED_ONE + GATED_QUARTERS)
def test_gated_calls_at_once_and_captured(gpu, n, hidden, cols, shape):
    torch = gpu
    _takes(shape, True, n, hidden, cols)
    w = _weights(torch, q4_0(n, 2 * hidden, cols)[0])
    ins = [_rows8(torch, n + i, n, cols)[2:] for i in range(2)]
    _at_once_and_captured(torch, lambda i, outs: w.gated(*ins[i], outs[1], outs[2], out=outs[0],
                                                         stream=torch.cuda.current_stream()),
                          lambda: (torch.zeros(n, hidden, device="cuda"),
                                   torch.zeros(n, hidden, dtype=torch.int8, device="cuda"),
                                   torch.zeros(n, hidden // 32, dtype=torch.float16, device="cuda")))


def _at_once_and_captured(torch, call, outputs):
    """call(i, outputs) for two inputs: one after another, on two streams at once, and replayed."""
    want = [outputs() for _ in range(2)]
    for i in range(2):
        call(i, want[i])
    torch.cuda.synchronize()
    assert not torch.equal(want[0][0], want[1][0])

    def equal(got):
        torch.cuda.synchronize()
        return all(torch.equal(g, t) for a, b in zip(got, want) for g, t in zip(a, b))

    got, streams = [outputs() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            call(i, got[i])
    assert equal(got)
    got, graph = [outputs() for _ in range(2)], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(2):
            call(i, got[i])
    for _ in range(3):
        for t in (*got[0], *got[1]):
            t.zero_()
        graph.replay()
        assert equal(got)

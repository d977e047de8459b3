"""Products of 8-bit rows with Q4_0 weights, plain and gated, against 64 bits."""
import numpy as np
import pytest

from _shapes import product_shapes
from _rows import blocks_of, check, check8, gated, product, q4_0, rounded, split8

pytestmark = pytest.mark.gpu


def _weights(torch, blocks, parts=1):
    from bmo_jetson_amd import Q4Weights
    rows, nb, _ = blocks.shape
    w = Q4Weights(rows, nb * 32)
    t = torch.from_numpy(blocks).cuda()
    cuts = [rows * i // parts for i in range(parts + 1)]
    for a, b in zip(cuts, cuts[1:]):
        w.load(t[a:b], row=a, stream=torch.cuda.current_stream())
    return w


def _rows8(torch, seed, n, cols):
    r = np.random.default_rng(seed)
    codes, scales = split8((r.standard_normal((n, cols)) * np.exp(r.standard_normal((1, cols)))).astype(np.float32))
    return codes, scales, torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()


def _product(torch, n, rows, cols, type_="float32", seed=0, parts=1):
    blocks, wc, ws = q4_0(seed, rows, cols)
    w = _weights(torch, blocks, parts)
    codes, scales, c, s = _rows8(torch, seed + 1, n, cols)
    out = torch.full((n + 1, rows), 7.0, dtype=getattr(torch, type_), device="cuda")
    w.product(c, s, out[:n], stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    ref, bound = product(codes, scales, wc, ws)
    check(out[:n].double().cpu().numpy(), ref, rounded(bound, ref, type_), f"{n} x {rows} x {cols} {type_}")
    assert (out[n] == 7).all()  # the row behind the last
    return w, codes, scales, c, s, wc, ws


ROWS = [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 513]


@pytest.mark.parametrize("n", ROWS)
def test_numbers_of_rows(gpu, n):
    _product(gpu, n, 160, 256, seed=n)
    _product(gpu, n, 96, 1120, "bfloat16", seed=n + 1)


@pytest.mark.parametrize("rows", [1, 3, 15, 16, 17, 31, 33, 64, 65, 130, 257, 1000])
def test_numbers_of_outputs(gpu, rows):
    for n in (1, 20, 70, 260):
        _product(gpu, n, rows, 192, seed=rows)


@pytest.mark.parametrize("cols", [32, 64, 96, 128, 160, 416, 992, 1024, 1056, 4096, 4128, 11264])
def test_numbers_of_columns(gpu, cols):
    for n in (1, 18, 66, 270):
        _product(gpu, n, 48, cols, seed=cols)


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,rows,cols", [(1, 4096, 4096), (5, 1001, 512), (40, 2050, 640), (150, 515, 1024), (700, 384, 512)])
def test_types_and_larger_sizes(gpu, n, rows, cols, type_):
    _product(gpu, n, rows, cols, type_)


# rows, outputs, columns and the kernel that takes them (workgroup's rows, outputs; waves of a piece)
SHAPES = [(2, 97, 416, (16, 16, 8)), (37, 161, 1120, (16, 16, 8)), (69, 1001, 1120, (16, 32, 8)), (33, 2001, 1120, (16, 32, 8)),
          (37, 4097, 416, (16, 32, 8)), (37, 4097, 1120, (16, 64, 8)), (2, 8193, 1120, (16, 64, 8)),
          (17, 8161, 1248, (32, 32, 4)), (197, 1001, 96, (32, 32, 4)), (325, 1057, 1120, (32, 32, 4)),
          (131, 1001, 736, (32, 32, 8)), (131, 1001, 2976, (32, 32, 8)), (49, 4001, 4000, (32, 32, 8)),
          (69, 8193, 416, (32, 64, 4)), (1501, 513, 416, (32, 64, 4)), (131, 4097, 2080, (32, 64, 4)),
          (131, 6001, 736, (32, 128, 1)), (901, 2049, 96, (32, 128, 1)), (261, 6001, 416, (32, 128, 1)),
          (261, 4097, 96, (32, 256, 1)), (515, 6001, 1120, (32, 256, 1)), (901, 4097, 1120, (32, 256, 1)),
          (515, 6001, 4000, (64, 128, 2)), (901, 4097, 4064, (64, 128, 2)),
          (901, 8193, 96, (64, 256, 1)), (515, 12001, 1120, (64, 256, 1)), (3001, 2049, 1120, (64, 256, 1))]
GATED_SHAPES = [(2, 32, 736, (16, 32, 8)), (261, 32, 2080, (16, 32, 8)), (2, 32, 96, (16, 32, 8)), (69, 160, 416, (16, 32, 8)),
                (131, 1024, 736, (32, 32, 8)), (69, 2080, 2080, (32, 32, 8)), (29, 6016, 4000, (32, 32, 8)),
                (131, 1024, 96, (32, 32, 4)), (69, 2080, 160, (32, 32, 4)), (37, 6016, 96, (32, 32, 4)),
                (901, 736, 736, (32, 64, 2)), (131, 4128, 32, (32, 64, 2)), (901, 4128, 96, (32, 128, 1)),
                (515, 2080, 736, (32, 128, 1)), (515, 3104, 2080, (64, 64, 2)), (1501, 1056, 2080, (64, 64, 2)),
                (1101, 3104, 736, (64, 128, 1)), (515, 6016, 1120, (64, 128, 1)), (1501, 2080, 1120, (64, 128, 1))]


@pytest.mark.parametrize("n,rows,cols,shape", SHAPES)
def test_every_kernel(gpu, n, rows, cols, shape):
    assert product_shapes([(False, n, rows, cols)]) == [shape]
    _product(gpu, n, rows, cols, seed=n)


@pytest.mark.parametrize("n,rows,cols,shape", SHAPES)
def test_every_kernel_s_stores(gpu, n, rows, cols, shape):
    """16-bit results are the 32-bit ones rounded, at every alignment of their
    rows; what lies between the rows stays."""
    torch = gpu
    blocks, _, _ = q4_0(n + 1, rows, cols)
    w = _weights(torch, blocks)
    _, _, c, s = _rows8(torch, n, n, cols)
    want = torch.empty(n, rows, device="cuda")
    stream = torch.cuda.current_stream()
    w.product(c, s, want, stream=stream)
    for type_ in (torch.float16, torch.bfloat16, torch.float32):
        for stride, shift in ((rows + (rows & 1), 0), (rows + 7, 0), (rows + 6 + (rows & 1), 2), (rows + 6, 1)):
            big = torch.full((n, stride), 7.0, dtype=type_, device="cuda")
            w.product(c, s, big[:, shift:shift + rows], stream=stream)
            assert torch.equal(big[:, shift:shift + rows], want.to(type_)), (type_, stride, shift)
            assert (big[:, :shift] == 7).all() and (big[:, shift + rows:] == 7).all()


def test_gemv_of_each_row(gpu):
    """A row's product is what the GEMV gives for it, but for the rounding of
    that one's block sums to fp16 and its scales to the nearest fp16."""
    torch = gpu
    from bmo_jetson_amd import Q4Weights, gemv_q4_0_q8_1, quantize_rows
    blocks, _, _ = q4_0(5, 512, 1024)
    t = torch.from_numpy(blocks).cuda()
    w = Q4Weights(512, 1024)
    w.load(t, stream=torch.cuda.current_stream())
    x = torch.randn(3, 1024, device="cuda")
    c, s = torch.empty(3, 1024, dtype=torch.int8, device="cuda"), torch.empty(3, 32, dtype=torch.float16, device="cuda")
    out, one = torch.empty(3, 512, device="cuda"), torch.empty(512, device="cuda")
    quantize_rows(x, c, s, stream=torch.cuda.current_stream())
    w.product(c, s, out, stream=torch.cuda.current_stream())
    for i in range(3):
        gemv_q4_0_q8_1(t, x[i], one, 512, 1024, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        # both quantize x to steps of amax / 127 within half a step
        step = (s[i].float() * 32**0.5).norm() * torch.from_numpy(np.abs(blocks[:, :, :2].copy().view(np.float16))).max().item()
        assert (out[i] - one).abs().max() <= 8 * step


def test_loaded_in_parts_strided_output(gpu):
    torch = gpu
    w, codes, scales, c, s, wc, ws = _product(torch, 37, 333, 384, parts=4)
    ref, bound = product(codes, scales, wc, ws)
    for type_ in ("float32", "float16"):
        for width, shift in ((340, 0), (341, 1), (336, 2), (333, 0)):
            big = torch.full((37, width), 7.0, dtype=getattr(torch, type_), device="cuda")
            w.product(c, s, big[:, shift:shift + 333], stream=torch.cuda.current_stream())
            torch.cuda.synchronize()
            check(big[:, shift:shift + 333].double().cpu().numpy(), ref, rounded(bound, ref, type_), "strided")
            assert (big[:, :shift] == 7).all() and (big[:, shift + 333:] == 7).all()
    from bmo_jetson_amd import RingError
    with pytest.raises(RingError, match="out of range"):
        w.load(torch.zeros(2, 12, 18, dtype=torch.uint8, device="cuda"), row=332)


@pytest.mark.parametrize("n", [1, 20, 40, 130, 300])
def test_extreme_codes_and_scales(gpu, n):
    """Every code at its end, scales from fp16's largest to its subnormals,
    signs mixed; a NaN or infinite scale spoils its own row or column only."""
    torch = gpu
    r = np.random.default_rng(n)
    rows, cols = 80, 320
    wc = r.choice([0, 15, 8], (rows, cols // 32, 32)).astype(np.uint8)
    wc[3], wc[4] = 0, 15
    ws = r.choice([65504.0, -65504.0, 2.0**-24, 1.0, 0.0, -0.0], (rows, cols // 32)).astype(np.float16)
    codes = r.choice([-127, 127, -128, 0, 1], (n, cols)).astype(np.int8)
    codes[0] = 127
    scales = r.choice([65504.0, 2.0**-24, 0.5, 0.0], (n, cols // 32)).astype(np.float16)
    ws[7, 2], ws[9, 9], scales[n // 2, 1], scales[n - 1, 9] = np.nan, np.inf, np.nan, np.inf
    w = _weights(torch, blocks_of(wc, ws))
    out = torch.empty(n, rows, device="cuda")
    w.product(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), out, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    spoiled = np.zeros((n, rows), bool)
    spoiled[[n // 2, n - 1]], spoiled[:, [7, 9]] = True, True
    ref, bound = product(codes, scales, wc, ws)
    assert np.isfinite(got[~spoiled]).all()
    check(np.where(spoiled, 0, got), np.where(spoiled, 0, ref), np.where(spoiled, 0, bound), "extreme")
    assert np.isnan(got[n // 2]).all() and np.isnan(got[:, 7]).all()


@pytest.mark.parametrize("n", [1, 5, 100])
@pytest.mark.parametrize("cols", [32, 96, 160])
def test_an_infinite_scale_in_the_last_block(gpu, n, cols):
    """What lies past the last block adds nothing, whatever that block's scale."""
    torch = gpu
    wc = np.full((40, cols // 32, 32), 9, np.uint8)
    w = _weights(torch, blocks_of(wc, np.full((40, cols // 32), -2.0, np.float16)))
    scales = np.ones((n, cols // 32), np.float16)
    scales[n // 2, -1] = np.inf
    out = torch.empty(n, 40, device="cuda")
    w.product(torch.ones(n, cols, dtype=torch.int8, device="cuda"), torch.from_numpy(scales).cuda(), out,
              stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert (out[n // 2] == -np.inf).all() and torch.isfinite(torch.cat((out[:n // 2], out[n // 2 + 1:]))).all()


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("n,hidden,cols", [c[:3] for c in GATED_SHAPES] + [
                                           (1, 32, 32), (1, 1056, 416), (7, 64, 256), (16, 96, 1024), (17, 512, 96), (33, 32, 640),
                                           (64, 160, 256), (65, 288, 256), (129, 64, 512), (300, 96, 160), (2, 5632, 4096)])
def test_gated(gpu, n, hidden, cols, activation):
    torch = gpu
    assert (n, hidden, cols, product_shapes([(True, n, hidden, cols)])[0]) in GATED_SHAPES or (n, hidden, cols) not in [
        c[:3] for c in GATED_SHAPES]
    blocks, wc, ws = q4_0(n, 2 * hidden, cols)
    ws = (ws.astype(np.float32) * 3).astype(np.float16)
    w = _weights(torch, blocks_of(wc, ws))
    codes, scales, c, s = _rows8(torch, n + 1, n, cols)
    both, off = product(codes, scales, wc, ws)
    h, bound = gated(both[:, :hidden], both[:, hidden:], off[:, :hidden], off[:, hidden:], activation)
    oc = torch.full((n + 1, hidden), 77, dtype=torch.int8, device="cuda")
    os = torch.full((n + 1, hidden // 32), 7.0, dtype=torch.float16, device="cuda")
    stream = torch.cuda.current_stream()
    w.gated(c, s, oc[:n], os[:n], activation=activation, stream=stream)
    torch.cuda.synchronize()
    check8(oc[:n].cpu().numpy(), os[:n].cpu().numpy(), h, bound, f"gated {n} {hidden} {cols}")
    assert (oc[n] == 77).all() and (os[n] == 7).all()
    for type_ in ("float32", "bfloat16"):  # with both kinds of output, and the other alone
        out = torch.empty(n, hidden, dtype=getattr(torch, type_), device="cuda")
        oc2, os2 = torch.zeros_like(oc[:n]), torch.zeros_like(os[:n])
        w.gated(c, s, oc2, os2, out=out, activation=activation, stream=stream)
        torch.cuda.synchronize()
        check(out.double().cpu().numpy(), h, rounded(bound, h, type_), "out")
        assert torch.equal(oc2, oc[:n]) and torch.equal(os2, os[:n])
        alone = torch.empty_like(out)
        w.gated(c, s, out=alone, activation=activation, stream=stream)
        assert torch.equal(alone, out)


def test_gated_far_out(gpu):
    """Gates so large that exp overflows, results past 8 bits' scales, NaN."""
    torch = gpu
    n, hidden, cols = 18, 64, 64
    wc = np.full((2 * hidden, 2, 32), 9, np.uint8)
    ws = np.full((2 * hidden, 2), 1.0, np.float16)
    ws[1::2] = -1.0
    w = _weights(torch, blocks_of(wc, ws))
    codes = np.full((n, cols), 100, np.int8)
    scales = np.ones((n, 2), np.float16)
    scales[1], scales[2], scales[3, 0], scales[4] = 0.0, 60000.0, np.nan, 2.0**-24
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    both, off = product(codes, scales, wc, ws)
    for activation in ("silu", "gelu"):
        h, bound = gated(both[:, :hidden], both[:, hidden:], off[:, :hidden], off[:, hidden:], activation)
        out = torch.empty(n, hidden, device="cuda")
        oc = torch.empty(n, hidden, dtype=torch.int8, device="cuda")
        os = torch.empty(n, 2, dtype=torch.float16, device="cuda")
        w.gated(c, s, oc, os, out=out, activation=activation, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        assert np.isnan(got[3]).all() and os[3].isnan().all() and not oc[3].any()
        rest = [i for i in range(n) if i != 3]
        check(got[rest], h[rest], rounded(bound, h, "float32")[rest], activation)
        check8(oc.cpu().numpy()[rest], os.cpu().numpy()[rest], h[rest], bound[rest], activation)
    from bmo_jetson_amd import RingError
    odd = _weights(torch, blocks_of(wc[:96], ws[:96]))
    with pytest.raises(RingError, match="whole blocks"):
        odd.gated(c, s, out=torch.empty(n, 48, device="cuda"))
    empty = torch.empty(0, hidden, device="cuda")
    w.gated(c[:0], s[:0], out=empty)
    w.product(c[:0], s[:0], torch.empty(0, 2 * hidden, device="cuda"))


def test_two_streams_and_captured(gpu):
    torch = gpu
    blocks, _, _ = q4_0(1, 256, 512)
    w = _weights(torch, blocks)
    torch.cuda.synchronize()
    for n in (1, 24, 80, 300):
        _, _, c, s = _rows8(torch, n, n, 512)
        want = torch.empty(n, 256, device="cuda")
        w.product(c, s, want, stream=torch.cuda.current_stream())
        oc, os = torch.empty(n, 128, dtype=torch.int8, device="cuda"), torch.empty(n, 4, dtype=torch.float16, device="cuda")
        w.gated(c, s, oc, os, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        outs = [torch.empty(n, 256, device="cuda") for _ in range(2)]
        for o in outs:  # two calls at once
            w.product(c, s, o, stream=torch.cuda.Stream())
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        o, oc2, os2 = torch.empty_like(want), torch.empty_like(oc), torch.empty_like(os)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.product(c, s, o, stream=torch.cuda.current_stream())
            w.gated(c, s, oc2, os2, stream=torch.cuda.current_stream())
        for _ in range(3):
            o.zero_(), oc2.zero_(), os2.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want) and torch.equal(oc2, oc) and torch.equal(os2, os)

"""RMS norm and 8-bit rows against 64 bits."""
import numpy as np
import pytest

from _rows import U, check, check8, rounded, scale8, split8, tensor

pytestmark = pytest.mark.gpu


def _rows(seed, n, dim):
    r = np.random.default_rng(seed)
    return (r.standard_normal((n, dim)) * np.exp(0.5 * r.standard_normal(dim))).astype(np.float32)


def _norm(torch, x, res, w, eps, out_type, codes, x_type="float32", r_type="float32", w_type="float32"):
    from bmo_jetson_amd import rms_norm
    n, dim = x.shape
    tx, x64 = tensor(torch, x, x_type)
    tw, w64 = tensor(torch, w, w_type)
    tr, r64 = (None, None) if res is None else tensor(torch, res, r_type)
    out = torch.full((n, dim), 7.0, dtype=getattr(torch, out_type), device="cuda") if out_type else None
    c = torch.full((n, dim), 77, dtype=torch.int8, device="cuda") if codes else None
    s = torch.full((n, dim // 32), 7.0, dtype=torch.float16, device="cuda") if codes else None
    rms_norm(tx, tw, eps, residual=tr, out=out, codes=c, scales=s, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    h = x64
    if res is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            h = torch.from_numpy(x64.astype(np.float32) + r64.astype(np.float32)).to(tr.dtype).double().numpy()
        np.testing.assert_array_equal(tr.double().cpu().numpy(), h)
    with np.errstate(invalid="ignore", over="ignore"):
        y = h / np.sqrt((h * h).sum(axis=1, keepdims=True) / dim + eps) * w64
    # squares sum up in at most 8 * 4 steps of a lane, 6 of a wave and 16 of waves, all of one sign, halved by the root;
    # the mean, its root, the quotient and two products
    off = np.abs(y) * (27 + 6) * U
    if out is not None:
        check(out.double().cpu().numpy(), y, rounded(off, y, out_type), "out")
    if codes:
        check8(c.cpu().numpy(), s.cpu().numpy(), y, off, "8-bit rows")
    return tx, tr, out, c, s


@pytest.mark.parametrize("n,dim", [(1, 4096), (3, 32), (5, 512), (2, 544), (70, 1024), (9, 2048), (4, 2080), (300, 4096),
                                   (2, 4128), (3, 8192), (2, 16384), (1, 16416), (2, 32768)])
def test_both_outputs(gpu, n, dim):
    w = np.random.default_rng(1).uniform(0.2, 2, dim)
    _norm(gpu, _rows(n, n, dim), _rows(n + 1, n, dim), w, 1e-5, "float32", True)


@pytest.mark.parametrize("n,dim", [(1, 1), (2, 7), (3, 33), (5, 155), (2, 1000), (2, 2047), (3, 4097), (1, 32767)])
def test_odd_sizes(gpu, n, dim):
    w = np.random.default_rng(1).uniform(-2, 2, dim)
    _norm(gpu, _rows(n, n, dim), None, w, 1e-6, "float32", False)
    _norm(gpu, _rows(n, n, dim), _rows(n + 1, n, dim), w, 1e-6, "bfloat16", False, "bfloat16", "float16", "float16")


@pytest.mark.parametrize("x_type", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("r_type", [None, "float32", "float16", "bfloat16"])
@pytest.mark.parametrize("out_type", ["", "float32", "float16", "bfloat16"])
def test_types(gpu, x_type, r_type, out_type):
    x, w = _rows(3, 6, 2080), np.random.default_rng(1).uniform(0.2, 2, 2080)
    res = None if r_type is None else 5 * _rows(4, 6, 2080)
    for w_type in ("float32", "float16", "bfloat16"):
        _norm(gpu, x, res, w, 1e-5, out_type, True, x_type, r_type or "float32", w_type)


def test_strides_alignment_and_in_place(gpu):
    torch = gpu
    from bmo_jetson_amd import rms_norm
    w = torch.rand(161, device="cuda") + 0.5
    for dim, shift in ((160, 0), (160, 1), (159, 2), (160, 8)):
        big = torch.randn(5, 3, 170, device="cuda")
        for type_ in (torch.float32, torch.float16):
            b = big.to(type_)
            x, res, out = b[:, 0, shift:shift + dim], b[:, 1, shift:shift + dim], b[:, 2, :dim]
            h = (x.float() + res.float()).to(type_).double()
            y = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5) * w[1:dim + 1].double()
            before = b.clone()
            rms_norm(x, w[1:dim + 1], residual=res, out=out, stream=torch.cuda.current_stream())
            torch.cuda.synchronize()
            off = (y.abs() * 33 * U).cpu().numpy()
            check(out.double().cpu().numpy(), y.cpu().numpy(), rounded(off, y.cpu().numpy(), str(type_)[6:]), "strided")
            assert torch.equal(res.double(), h)
            assert torch.equal(b[:, 0], before[:, 0]) and torch.equal(b[:, 1, :shift], before[:, 1, :shift])
            assert torch.equal(b[:, 1, shift + dim:], before[:, 1, shift + dim:])
            assert torch.equal(b[:, 2, dim:], before[:, 2, dim:])
            x2 = x.clone()
            rms_norm(x2, w[1:dim + 1], out=x2, stream=torch.cuda.current_stream())  # in place
            out2 = torch.empty_like(x2)
            rms_norm(x, w[1:dim + 1], out=out2, stream=torch.cuda.current_stream())
            assert torch.equal(x2, out2)


def test_rows_that_are_not_finite_and_rows_of_zeros(gpu):
    torch = gpu
    x = _rows(5, 8, 4096)
    x[1, 77], x[2, 5], x[3, 9], x[5] = np.nan, np.inf, -np.inf, 0
    w = np.ones(4096)
    _, _, out, c, s = _norm(torch, x[[0, 4, 5, 6]], None, w, 1e-5, "float32", True)
    assert not out[2].any() and not c[2].any() and not s[2].any()
    from bmo_jetson_amd import rms_norm
    c = torch.empty(8, 4096, dtype=torch.int8, device="cuda")
    s = torch.empty(8, 128, dtype=torch.float16, device="cuda")
    out = torch.empty(8, 4096, device="cuda")
    rms_norm(tensor(torch, x, "float32")[0], torch.ones(4096, device="cuda"), out=out, codes=c, scales=s,
             stream=torch.cuda.current_stream())
    # a NaN spoils its row; an infinity makes its own element NaN (inf / inf) and its row's others zeros
    assert torch.isnan(out[1]).all() and torch.isnan(s[1].float()).all() and not c[1].any()
    for r, at in ((2, 5), (3, 9)):
        assert torch.isnan(out[r, at]) and torch.isnan(s[r, at // 32].float()) and not c[r].any()
    assert torch.isfinite(out[[0, 4, 5, 6, 7]]).all()


def test_eps_alone_and_no_rows(gpu):
    torch = gpu
    from bmo_jetson_amd import quantize_rows, rms_norm
    x = np.full((2, 64), 1e-20, dtype=np.float32)
    _norm(torch, x, None, np.ones(64), 1e-5, "float32", True)
    e = torch.empty(0, 64, device="cuda")
    c, s = torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, 2, dtype=torch.float16, device="cuda")
    rms_norm(e, torch.ones(64, device="cuda"), out=e, codes=c, scales=s)
    quantize_rows(e, c, s)


@pytest.mark.parametrize("type_", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,cols", [(1, 32), (3, 96), (70, 4096), (9, 11264), (513, 1024)])
def test_quantize_rows(gpu, n, cols, type_):
    torch = gpu
    from bmo_jetson_amd import quantize_rows
    x = _rows(n, n, cols + 8)
    t, x64 = tensor(torch, x, type_)
    for view, v64 in ((t[:, :cols].contiguous(), x64[:, :cols]), (t[:, 3:cols + 3], x64[:, 3:cols + 3])):
        c = torch.empty(n, cols, dtype=torch.int8, device="cuda")
        s = torch.empty(n, cols // 32, dtype=torch.float16, device="cuda")
        quantize_rows(view, c, s, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        check8(c.cpu().numpy(), s.cpu().numpy(), v64, 0.0, "rows")
        np.testing.assert_array_equal(s.cpu().numpy(), split8(v64)[1])  # scales are exact


def test_quantize_blocks_at_the_ends_of_the_range(gpu):
    torch = gpu
    from bmo_jetson_amd import quantize_rows
    top = np.float32(127 * 65504.0)
    firsts = [0.0, 1e-45, 1e-30, 2.0**-24 * 127, 2.0**-24 * 127.5, 1e-3, 127 * 1.00001, top, np.nextafter(top, np.float32(1e9)),
              1e30, np.inf, np.nan, -np.inf, -top]
    x = np.zeros((len(firsts), 64), dtype=np.float32)
    x[:, 3] = firsts
    x[:, 40] = 1.0  # the block beside is not touched
    with np.errstate(invalid="ignore"):
        x[:, 4] = x[:, 3] * np.float32(-0.5)
    x[~np.isfinite(x[:, 3]), 4] = 3.0
    c = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    s = torch.empty(len(firsts), 2, dtype=torch.float16, device="cuda")
    quantize_rows(torch.from_numpy(x).cuda(), c, s, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    check8(c.cpu().numpy(), s.cpu().numpy(), x.astype(np.float64), 0.0, "ends")
    np.testing.assert_array_equal(s.cpu().numpy()[:, 0], scale8(np.abs(x[:, 3])))
    np.testing.assert_array_equal(s.cpu().numpy()[:, 1], scale8(np.float32(1)))


def test_captured_and_on_another_stream(gpu):
    torch = gpu
    from bmo_jetson_amd import rms_norm
    x, res = torch.randn(5, 1024, device="cuda"), torch.zeros(5, 1024, device="cuda")
    w, out = torch.rand(1024, device="cuda"), torch.empty(5, 1024, device="cuda")
    c, s = torch.empty(5, 1024, dtype=torch.int8, device="cuda"), torch.empty(5, 32, dtype=torch.float16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        rms_norm(x, w, residual=res, out=out, codes=c, scales=s, stream=torch.cuda.current_stream())
    for i in range(4):
        x.normal_()
        want = res + x
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(res, want), i
        y = torch.empty_like(out)
        rms_norm(want, w, out=y, stream=torch.cuda.current_stream())
        assert torch.equal(y, out), i

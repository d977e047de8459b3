"""Rows whose offsets pass 32 bits, and columns past what one row keeps in LDS:
the rows at both ends against 64 bits (by the helper's oracle), all others
against the same rows elsewhere."""
import numpy as np
import pytest

from _rows import blocks_of, check, check8, product, q4_0, rounded, split8

pytestmark = pytest.mark.gpu


def _weights(torch, seed, rows, cols):
    from bmo_jetson_amd import Q4Weights
    _, wc, ws = q4_0(seed, rows, cols)
    w = Q4Weights(rows, cols)
    w.load(torch.from_numpy(blocks_of(wc, ws)).cuda(), stream=torch.cuda.current_stream())
    return w, wc, ws


@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("cols", [32768, 32800, 33600])
def test_long_rows(gpu, n, cols):
    torch = gpu
    w, wc, ws = _weights(torch, cols, 64, cols)
    codes, scales = split8(np.random.default_rng(n).standard_normal((n, cols)).astype(np.float32))
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    out, half = torch.empty(n, 64, device="cuda"), torch.empty(n, 32, device="cuda")
    w.product(c, s, out, stream=torch.cuda.current_stream())
    w.gated(c, s, out=half, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    ref, bound = product(codes, scales, wc, ws)
    check(out.double().cpu().numpy(), ref, rounded(bound, ref, "float32"), f"{n} x {cols}")
    # the activation of the plain product's outputs: both sums are off by the bound, the gate's slope is below 1.1,
    # and exp, the division and the products round a dozen times
    g, u = out[:, :32].double().cpu().numpy(), out[:, 32:].double().cpu().numpy()
    want, b = g / (1 + np.exp(-g)) * u, bound
    slack = 2 * (1.1 * b[:, :32] * (np.abs(u) + b[:, 32:]) + (np.abs(g) + b[:, :32]) * b[:, 32:]) + 16 * 2.0**-24 * np.abs(want)
    assert (np.abs(half.double().cpu().numpy() - want) <= slack + 1e-30).all()


def _repeated(torch, n, cols, period=97):
    """n rows of `period` different ones in turn, as 8-bit rows."""
    codes, scales = split8(np.random.default_rng(5).standard_normal((period, cols)).astype(np.float32))
    at = torch.arange(n, device="cuda") % period
    return codes, scales, torch.from_numpy(codes).cuda()[at], torch.from_numpy(scales).cuda()[at], at


def _same(torch, got, first, at, step=65536):
    for i in range(0, got.shape[0], step):
        assert torch.equal(got[i:i + step], first[at[i:i + step]]), f"rows from {i}"


def test_codes_past_32_bits(gpu):
    """2^20 rows of 4128 codes: 4.3 G of them."""
    torch = gpu
    n, cols = 1 << 20, 4128
    w, wc, ws = _weights(torch, 1, 64, cols)
    codes, scales, c, s, at = _repeated(torch, n, cols)
    out = torch.empty(n, 64, device="cuda", dtype=torch.bfloat16)
    oc, os = torch.empty(n, 32, device="cuda", dtype=torch.int8), torch.empty(n, 1, device="cuda", dtype=torch.float16)
    w.product(c, s, out, stream=torch.cuda.current_stream())
    w.gated(c, s, oc, os, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    ref, bound = product(codes, scales, wc, ws)
    check(out[:97].double().cpu().numpy(), ref, rounded(bound, ref, "bfloat16"), "first rows")
    for got in (out, oc, os):
        _same(torch, got, got[:97].clone(), at)


def test_outputs_past_32_bits(gpu):
    """70001 rows of 65600 outputs: 4.6 G of them; and of half as many, gated."""
    torch = gpu
    n, rows = 70001, 65600
    w, wc, ws = _weights(torch, 2, rows, 32)
    codes, scales, c, s, at = _repeated(torch, n, 32)
    out = torch.empty(n, rows, device="cuda", dtype=torch.float16)
    w.product(c, s, out, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    ref, bound = product(codes, scales, wc, ws)
    check(out[:97].double().cpu().numpy(), ref, rounded(bound, ref, "float16"), "first rows")
    _same(torch, out, out[:97].clone(), at, 4096)
    oc = torch.empty(n, rows // 2, device="cuda", dtype=torch.int8)
    os = torch.empty(n, rows // 64, device="cuda", dtype=torch.float16)
    w.gated(c, s, oc, os, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    for got in (oc, os):
        _same(torch, got, got[:97].clone(), at, 4096)


def test_norm_quantize_and_rope_past_32_bits(gpu):
    """140001 rows of 32768 values: 4.6 G of them."""
    torch = gpu
    from bmo_jetson_amd import Rope, quantize_rows, rms_norm
    n, dim = 140001, 32768
    stream = torch.cuda.current_stream()
    at = torch.arange(n, device="cuda") % 97
    base = torch.randn(97, dim, device="cuda").half()
    x = base[at]
    weight = torch.rand(dim, device="cuda")
    c, s = torch.empty(n, dim, dtype=torch.int8, device="cuda"), torch.empty(n, dim // 32, dtype=torch.float16, device="cuda")
    quantize_rows(x, c, s, stream=stream)
    torch.cuda.synchronize()
    values = base.float().cpu().numpy()
    # (scales are exact; a code may be the other neighbour where x / d is halfway: x * (1 / d) rounds twice)
    assert np.array_equal(s[:97].cpu().numpy(), split8(values)[1])
    check8(c[:97].cpu().numpy(), s[:97].cpu().numpy(), values.astype(np.float64), 0.0, "first rows")
    _same(torch, c, c[:97].clone(), at, 4096)
    _same(torch, s, s[:97].clone(), at)
    rms_norm(x, weight, out=x, codes=c, scales=s, stream=stream)
    few, fc, fs = torch.empty_like(base), c[:97].clone(), s[:97].clone()
    rms_norm(base, weight, out=few, codes=fc, scales=fs, stream=stream)
    torch.cuda.synchronize()
    for got, first in ((x, few), (c, fc), (s, fs)):
        _same(torch, got, first, at, 4096)
    # 2^32 elements at most: 131072 tokens of 256 heads of 128 in place, at a stride of 40000 elements
    del c, s, x
    rope, tokens = Rope(128), 131072
    pos = at[:tokens].to(torch.int32)
    q = torch.empty(tokens, 40000, dtype=torch.float16, device="cuda")
    for i in range(0, tokens, 4096):
        q[i:i + 4096, :dim] = base[at[i:i + 4096]]
    rows = q[:, :dim].unflatten(1, (256, 128))
    rope.apply(pos, rows, stream=stream)
    first = base.clone().unflatten(1, (256, 128))
    rope.apply(torch.arange(97, dtype=torch.int32, device="cuda"), first, stream=stream)
    torch.cuda.synchronize()
    _same(torch, rows, first, at[:tokens], 4096)

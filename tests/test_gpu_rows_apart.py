"""Calls on rows that lie apart in one tensor: those that share bytes with what
is written are refused and leave it as it is, those that do not run."""
import pytest

import bmo_jetson_amd as bmo

pytestmark = pytest.mark.gpu


def _refused(torch, call, *tensors):
    before = [t.clone() for t in tensors]
    with pytest.raises(bmo.RingError, match="overlaps"):
        call()
    torch.cuda.synchronize()
    assert all(torch.equal(t, b) for t, b in zip(tensors, before))


def test_heads_of_one_packed_tensor(gpu):
    torch = gpu
    packed, pos = torch.randn(5, 6, 16, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")
    with bmo.Rope(16) as rope:
        _refused(torch, lambda: rope.apply(pos, packed[:, :2], q_out=packed[:, 1:3]), packed)
        _refused(torch, lambda: rope.apply(pos, packed[:, :2], packed[:, 1:3]), packed)
        _refused(torch, lambda: rope.apply(pos, packed[:, :2], packed[:, 4:], packed[:, 2:4], packed[:, 3:5]), packed)
        _refused(torch, lambda: rope.apply(packed.view(torch.int32)[4, 5, 11:], packed[:, 4:]), packed)
        want = torch.empty(5, 2, 16, device="cuda")
        rope.apply(pos, packed[:, :2], q_out=want, stream=torch.cuda.current_stream())
        rope.apply(pos, packed[:, :2], q_out=packed[:, 2:4], stream=torch.cuda.current_stream())
        assert torch.equal(packed[:, 2:4], want)


def test_columns_of_one_wide_tensor(gpu):
    torch = gpu
    big, w = torch.randn(3, 160, device="cuda"), torch.rand(64, device="cuda")
    other = torch.empty(3, 64, device="cuda")
    _refused(torch, lambda: bmo.rms_norm(big[:, 32:96], w, residual=big[:, :64], out=other), big)
    _refused(torch, lambda: bmo.rms_norm(big[:, 32:96], w, out=big[:, :64]), big)
    _refused(torch, lambda: bmo.rms_norm(other, big[1, 8:72], out=big[:, 64:128]), big)
    bmo.rms_norm(big[:, 64:128], w, out=other, stream=torch.cuda.current_stream())
    bmo.rms_norm(big[:, 64:128], w, out=big[:, :64], stream=torch.cuda.current_stream())
    assert torch.equal(big[:, :64], other)


def test_results_over_8_bit_rows(gpu):
    """Rows of 128 results, 1024 bytes apart in a buffer that holds the 8-bit rows too."""
    torch = gpu
    mem = torch.zeros(8192, dtype=torch.uint8, device="cuda")

    def at(a, shape, type_):
        size = torch.empty((), dtype=type_).element_size()
        n = shape[0] * shape[1]
        return mem[a:a + n * size].view(type_).view(shape)

    out = at(0, (4, 256), torch.float32)[:, :128]
    away = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, dtype=torch.float16, device="cuda")
    stream = torch.cuda.current_stream()
    with bmo.Q4Weights(128, 64) as w, bmo.Q4Weights(256, 64) as g:
        for a in (1024 - 240, 1024, 1024 + 496, 3 * 1024 + 496):
            _refused(torch, lambda: w.product(at(a, (4, 64), torch.int8), away[1], out, stream=stream), mem)
        for a in (1024 - 14, 1024, 1024 + 510):
            _refused(torch, lambda: w.product(away[0], at(a, (4, 2), torch.float16), out, stream=stream), mem)
        _refused(torch, lambda: g.gated(*away, out=out, out_codes=at(0, (4, 128), torch.int8),
                                        out_scales=at(4096, (4, 4), torch.float16), stream=stream), mem)
        for a in (512, 1024 - 256, 3 * 1024 + 512):  # between the rows
            w.product(at(a, (4, 64), torch.int8), away[1], out, stream=stream)
        torch.cuda.synchronize()
        assert not mem.any()

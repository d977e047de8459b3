"""Which tensors of a call share bytes, and that calls on rows which lie apart
are refused where they do, without a GPU."""
import os
import random
import subprocess

import pytest

import bmo_jetson_amd as bmo
from test_rows_abi import A, _norm

EXE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "build", "span_check")


def _meet(pairs):
    assert os.path.exists(EXE), "tests/build/span_check is not built (run __graft_entry__.build())"
    lines = "".join(" ".join(map(str, a + b)) + "\n" for a, b in pairs)
    out = subprocess.run([EXE], input=lines, capture_output=True, text=True, timeout=60, check=True).stdout.split()
    assert len(out) == len(pairs)
    return [o == "1" for o in out]


def _bytes(span):
    at, n, dense, stride = span
    return {at + i * stride + j for i in range(n) for j in range(dense)}


def test_small_spans():
    """Against the bytes themselves."""
    r = random.Random(5)

    def span(at):
        dense = r.choice([1, 2, 3, 4, r.randint(1, 20)])
        return (at, r.choice([1, 2, 3, r.randint(1, 30)]), dense, dense + r.choice([0, 1, 2, 5, r.randint(0, 60)]))

    pairs = [(span(2000), span(2000 + r.choice([0, 1, -1, 3, r.randint(-40, 40), r.randint(-900, 900)]))) for _ in range(6000)]
    pairs += [((2000, 9, d, s), (2000 + k, 9, e, s)) for s in (12, 13) for d in (1, 5, 7, 12) for e in (1, 6, 7) for k in range(-14, 15)]
    want = [bool(_bytes(a) & _bytes(b)) for a, b in pairs]
    assert 1000 < sum(want) < len(want) - 1000
    got = _meet(pairs)
    assert [p for p, g, w in zip(pairs, got, want) if g != w] == []
    assert _meet([(b, a) for a, b in pairs]) == want


def test_large_spans():
    """Rows and strides at the ends of their ranges; columns of one wide tensor."""
    far, top = 1 << 42, 1 << 30
    assert _meet([((4096, top, 64, far), (4096 + 64, top, 64, far)), ((4096, top, 65, far), (4096 + 64, top, 64, far)),
                  ((4096, top, 64, far), (4096 + far - 63, 1, 64, 64)), ((4096, top, 64, far), (4096 + far - 64, 1, 64, 64)),
                  # strides of different parity: the rows meet where one has come a whole stride nearer
                  ((4096, top, 1, far), (4096 + 1, top, 1, far - 1)), ((4096, 9, 1, far), (4096 + 9, 9, 1, far - 1)),
                  ((4096, top, 4, 1000), (4096 + 500, top, 4, 2000)), ((4096, top, 4, 1000), (4096 + 500, top, 4, 2004))]) == [
                      False, True, True, False, True, False, False, True]


def test_rows_between_rows():
    """Of different strides: each begins where one of the other's has ended."""
    assert _meet([((A, 2, 256, 512), (A + 256, 2, 256, 768)), ((A, 3, 128, 512), (A + 640, 3, 128, 256))]) == [False, False]


# (2 rows of 64 in fp32: 256 bytes each, 512 apart where the strides are 128)
@pytest.mark.parametrize("args", [
    dict(xs=128, out=A + 128, os=128), dict(xs=128, out=A + 508, os=128), dict(xs=128, res=A + 128, rs=128, out=A + 4096),
    dict(xs=128, res=A + 4096, rs=128, out=A + 4096 + 252, os=128), dict(xs=128, out=A + 512, os=64),
    dict(xs=128, out=A + 4096, os=128, w=A + 4096 + 512 + 252), dict(xs=128, out=A + 256, os=96),
    dict(xs=128, out=None, codes=A + 512, scales=A + 4096), dict(xs=128, out=None, codes=A + 256, scales=A + 764),
    dict(n=3, type=1, xs=256, out=A + 768, ot=1, os=128)])
def test_norm_refuses_rows_that_lie_apart(args):
    assert _norm(**{"w": A + 65536, "out": A + 32768, **args}) == 2
    assert "overlaps" in bmo.lib().bmo_rows_last_error().decode()


def test_quantize_refuses_rows_that_lie_apart():
    for x, stride, codes, scales in ((A, 128, A + 512, A + 4096), (A, 128, A + 4096, A + 508), (A + 64, 128, A, A + 4096)):
        assert bmo.lib().bmo_quantize_rows(2, 64, 0, x, stride, codes, scales, None) == 2
        assert "overlaps" in bmo.lib().bmo_rows_last_error().decode()

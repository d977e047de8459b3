"""Outputs that a call would leave as they are, without a GPU."""
import pytest

import bmo_jetson_amd as bmo


def test_rotary_keys_without_keys():
    torch = pytest.importorskip("torch")
    rope = bmo.Rope.__new__(bmo.Rope)
    rope._h, rope._device, rope.head_dim = None, -1, 16
    pos, q = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 16)
    with pytest.raises(ValueError, match="k_out without k"):
        rope.apply(pos, q, k_out=q)

"""The paged cache's C ABI without a GPU: refusals of create and NULL handles."""
import pytest

import bmo_jetson_amd as bmo


@pytest.mark.parametrize("args,why", [
    ((0, 1, 64, 1, 64), "positive"), ((1, 0, 64, 1, 64), "positive"), ((1, 1, 64, 0, 64), "positive"),
    ((1, 1, 64, 1, 96), "head_dim"), ((1, 1, 16, 1, 64), "page_size"), ((1, 1, 8, 1, 128), "page_size"),
    ((1, 1, 48, 1, 128), "page_size"), ((1, 1, 2048, 1, 128), "page_size"), ((1, 1, 0, 1, 128), "page_size"),
    ((1, 1 << 22, 1024, 1, 128), "2^31"), ((1 << 20, 1 << 20, 1024, 60000, 128), "large")])
def test_create_rejects_bad_geometry(args, why):
    L = bmo.lib()
    assert not L.bmo_kv_pages_create(*args)
    err = L.bmo_kv_pages_last_error(None).decode()
    assert err.startswith("bmo_kv_pages_create:")
    if why != "large":
        assert why in err
    with pytest.raises(RuntimeError, match="bmo_kv_pages_create failed"):
        bmo.KVPages(*args)


def test_null_handles():
    L = bmo.lib()
    L.bmo_kv_pages_free(None)
    assert L.bmo_kv_pages_bytes(None) == 0 and L.bmo_kv_pages_workspace_bytes(None, 4) == 0
    assert L.bmo_kv_pages_list_init(None, None, None) == 1
    assert L.bmo_kv_pages_plan(None, None, 1, None, None, None, 1, None, 0, None, None, None, None, None) == 1
    assert L.bmo_kv_pages_append(None, 0, 1, None, 0, None, None, 0, None) == 1
    assert L.bmo_kv_pages_gather(None, 0, 1, None, 0, None, None, 0, None) == 1
    assert L.bmo_kv_pages_decode(None, 0, 1, None, None, 1, 1, 0, None, 0, None, 0.0, 0, 0, None, 0, None) == 1
    assert L.bmo_kv_pages_append_decode(None, 0, 1, None, None, 1, 1, 0, None, 0, None, None, 0, None, 0.0, 0, 0, None, 0,
                                        None) == 1
    assert L.bmo_kv_pages_attend(None, 0, 1, None, None, None, 1, 1, 1, 1, None, 0, None, 0.0, 1, 0, 0, 0, None, 0,
                                 None) == 1


def _stand_in(device=-1):
    """A KVPages without a pool behind it: its checks of tensors, on the CPU."""
    from bmo_jetson_amd import KVPages
    p = KVPages.__new__(KVPages)
    p._h, p._device, p.n_pages, p.n_kv_heads, p.head_dim = None, device, 4, 2, 64
    return p


def test_tensors_that_are_refused():
    torch = pytest.importorskip("torch")
    p = _stand_in()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    lens, table, slots, q = i(3), i(3, 2), i(3), torch.zeros(3, 4, 64)
    row = torch.zeros(1, 2, 64).expand(3, 2, 64)  # the same row three times
    kv = torch.zeros(3, 2, 64)
    cases = [(lambda: p.decode(0, lens, table, q[:1].expand(3, 4, 64), q), "overlap"),
             (lambda: p.append(0, slots, row, kv), "overlap"),
             (lambda: p.gather(0, slots, kv, row), "overlap"),
             (lambda: p.append_decode(0, lens, table, q, row, row, q), "overlap"),
             (lambda: p.decode(0, lens, table, q, q, workspace=torch.zeros(64)[::2]), "workspace"),
             (lambda: p.decode(0, lens, i(2, 3).t(), q, q), "contiguous"),
             (lambda: p.decode(0, i(3).long(), table, q, q), "int32"),
             (lambda: p.attend(0, i(3), lens, table, q, q), "4 elements"),
             (lambda: p.plan(i(6), i(3), lens, table, slots=i(5), positions=i(4)), "same size"),
             (lambda: p.plan(i(5), i(3), lens, table), "6 elements")]
    for call, why in cases:
        with pytest.raises(ValueError, match=why):
            call()
    there = _stand_in(device=0)  # a pool on a GPU, tensors that are not
    for call in (lambda: there.decode(0, lens, table, q, q), lambda: there.append(0, slots, kv, kv),
                 lambda: there.list_init(i(6))):
        with pytest.raises(ValueError, match="device"):
            call()

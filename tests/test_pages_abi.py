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

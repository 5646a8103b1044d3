"""Arguments that the layers' products refuse before they look for a device."""
import pytest


def refused(match, f, *a):
    from systemds_amd import capi
    with pytest.raises(capi.ClaError, match=match) as e:
        f(*a)
    assert e.value.code == capi.ERR_INVALID


def test_quantize_rows():
    from systemds_amd import capi
    f, p = capi.quantize_rows_dev_async, 1 << 20
    refused("type 7", f, p, 7, 3, 8, 8, p, 8, p)
    refused("type -1", f, p, -1, 3, 8, 8, p, 8, p)
    refused("-2 rows", f, p, 0, -2, 8, 8, p, 8, p)
    refused("2147483648 rows", f, p, 0, 1 << 31, 8, 8, p, 8, p)
    refused("rows of 0 values", f, p, 0, 3, 0, 8, p, 8, p)
    refused("Y is null", f, None, 0, 3, 8, 8, p, 8, p)
    refused("Y is not aligned", f, p + 4, 0, 3, 8, 8, p, 8, p)
    refused("leading dimension 7 of Y", f, p, 0, 3, 8, 7, p, 8, p)
    refused("the 8-bit rows is null", f, p, 0, 3, 8, 8, None, 8, p)
    refused("leading dimension 7 of the 8-bit rows", f, p, 0, 3, 8, 8, p, 7, p)
    refused("the scales is null", f, p, 0, 3, 8, 8, p, 8, None)
    refused("the scales is not aligned", f, p, 0, 3, 8, 8, p, 8, p + 2)
    refused("leading dimension", f, p, 0, 3, 8, 1 << 62, p, 8, p)


def test_handles():
    from systemds_amd import capi
    lib = capi.load_library()
    for f in (lib.cla_q8_num_rows, lib.cla_q8_num_cols, lib.cla_q8_device_bytes):
        assert f(None) == capi.ERR_INVALID
    assert lib.cla_q8_workspace(None, 3) == capi.ERR_INVALID
    assert lib.cla_q8_lmm_dev_async(None, None, 0, 1, 1, None, None, 1, None, 0) == capi.ERR_INVALID
    assert b"null 8-bit matrix handle" in lib.cla_last_error()
    assert lib.cla_block_quantize_rows_dev_async(None, None, 8, None) == capi.ERR_INVALID
    lib.cla_q8_free(None)

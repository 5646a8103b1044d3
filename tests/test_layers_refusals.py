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
    refused("rows of 1073741825 values", f, p, 0, 3, (1 << 30) + 1, 1 << 31, p, 1 << 31, p)
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


def test_gate():
    from systemds_amd import capi
    p = 1 << 20
    names = ("act", "t", "y", "m", "k", "ldy", "w", "ldw", "b", "n")
    good = (1, 1, p, 3, 8, 8, p, 8, None, 4)

    def forward(out=p, ld=4, **kw):
        return [kw.get(x, v) for x, v in zip(names, good)] + [out, ld]
    for match, kw in [("activation 6", dict(act=6)), ("activation -1", dict(act=-1)), ("type 4", dict(t=4)), ("-1 rows", dict(m=-1)), ("weights of 0 x 4", dict(k=0)),
                      ("weights of 8 x 0", dict(n=0)), ("Y is null", dict(y=None)), ("Y is not aligned", dict(y=p + 2)), ("leading dimension 7 of Y", dict(ldy=7)),
                      ("W is null", dict(w=None)), ("leading dimension 7 of W", dict(ldw=7)), ("bias is not aligned", dict(b=p + 1)),
                      ("the output is null", dict(out=None)), ("leading dimension 3 of the output", dict(ld=3))]:
        refused(match, capi.gate_dev_async, *forward(**kw))

    def backward(d=p, ldd=4, gy=p, ldgy=8, gw=p, ldgw=8, gb=p, **kw):
        return [kw.get(x, v) for x, v in zip(names, good)] + [d, ldd, gy, ldgy, gw, ldgw, gb, p, 1 << 30]
    for match, kw in [("activation 9", dict(act=9)), ("incoming gradient is null", dict(d=None)), ("dimension 3 of the incoming", dict(ldd=3)),
                      ("dimension 7 of the gradient of Y", dict(ldgy=7)), ("dimension 7 of the gradient of W", dict(ldgw=7)), ("gradient of the bias", dict(gb=p + 1)),
                      ("no gradient is asked for", dict(gy=None, gw=None, gb=None)), ("Y is null", dict(y=None))]:
        refused(match, capi.gate_backward_dev_async, *backward(**kw))
    for kw in (dict(k=(4 << 20) // 4 + 1, ldy=1 << 21, ldw=1 << 21), dict(n=(1 << 20) // 4 + 1)):
        with pytest.raises(capi.ClaError, match="at most") as e:
            capi.gate_dev_async(*forward(ld=1 << 21, **kw))
        assert e.value.code == capi.ERR_UNSUPPORTED
    with pytest.raises(capi.ClaError, match="2 GiB"):
        capi.gate_dev_async(*forward(ldw=1 << 30))
    refused("type 5", capi.gate_workspace, 5, 3, 8, 4, True)
    refused("-3 rows", capi.gate_workspace, 1, -3, 8, 4, True)
    assert capi.gate_workspace(1, 100, 8, 4, False) == 0 == capi.gate_workspace(1, 0, 8, 4, True) < capi.gate_workspace(1, 1, 8, 4, True)

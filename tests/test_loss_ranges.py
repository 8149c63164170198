"""What the cross entropy takes and refuses at the ends of its ranges, and what it asks for in memory there. On the CPU: sizes and refusals touch no device."""
import ctypes as C

import pytest

from trips_amd import _lib, abi

F32, BF16, F16 = 0, 2, 3


def _desc(n, t, c, dtype=F32, scale=1.0):
    return abi.TripsTableLossDesc(abi.TRIPS_ABI_VERSION, dtype, abi.TRIPS_INDEX_I64, abi.TRIPS_REDUCE_MEAN, n, t, c, scale, c, c, c, c)


def _workspace(backward, *args, **kw):
    bytes_ = C.c_size_t(0)
    rc = _lib.load().trips_table_loss_workspace_size(C.byref(_desc(*args, **kw)), backward, C.byref(bytes_))
    return rc, bytes_.value


@pytest.mark.parametrize("scale,taken", [(2.35e38, True), (-2.35e38, True), (2.4e38, False), (-3.4e38, False), (1e-45, True), (0.0, True)])
def test_scales(scale, taken):
    """What the kernels multiply by is scale log2 e: infinite from 2.36e38 on."""
    rc, _ = _workspace(0, 10, 10, 8, scale=scale)
    assert rc == (abi.TRIPS_OK if taken else abi.TRIPS_ERR_INVALID_ARG)
    assert taken or b"scale" in _lib.load().trips_last_error_string()

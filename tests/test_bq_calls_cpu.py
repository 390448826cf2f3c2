"""The block quantiser's arguments and handles, as far as no device is needed."""
import ctypes as C

import pytest

from proxima_b200 import _native as N


def test_null_sessions_are_a_status_and_no_crash():
    lib = N.load()
    rows = N.PxcBqRows(None, None, 0, 16, 4)
    err = N.PxcError()
    r, e = C.byref(rows), C.byref(err)
    for status in (
        lib.pxc_bq_session_encode(None, None, 0, 8, 8, r, None, e),
        lib.pxc_bq_session_decode(None, r, 8, None, 0, 8, None, e),
        lib.pxc_bq_session_product(None, r, r, 8, None, 0, 8, None, e),
        lib.pxc_bq_session_grouped_product(None, r, None, r, None, 1, 8, None, 0, 0, None, e),
        lib.pxc_bq_session_report(None, e),
        lib.pxc_bq_session_check(None, None, e),
    ):
        assert status == 7 and err.parameter == b"session"
    handle = N.vp()
    assert lib.pxc_bq_session_create(None, C.byref(handle), e) == 7 and err.parameter == b"ctx"
    assert handle.value is None
    lib.pxc_bq_session_destroy(None)

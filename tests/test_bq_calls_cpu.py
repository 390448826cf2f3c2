"""The block quantiser's arguments and handles, as far as no device is needed."""
import ctypes as C

import numpy as np
import pytest

from proxima_b200 import _native as N
from proxima_b200.blockquant import BlockCodes, BlockQuantizer
from proxima_b200.errors import Configuration


class NoContext:
    """Stands for a context: nothing here reaches the device."""

    handle = None
    device = 0


def codes(n, dim):
    blocks = -(-dim // 128)
    return BlockCodes(np.zeros((n, -(-dim // 16) * 16), np.uint8), np.zeros((n, -(-blocks // 4) * 4), np.uint8), dim)


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


@pytest.mark.parametrize("bad", [[0, 1.5, 4], [0.0, 4.0], [[0, 1], [1, 4]], np.zeros((2, 0), np.int64), 4, ["0", "4"],
                                 [False, True]])
@pytest.mark.parametrize("side", [0, 1])
def test_host_offsets_that_are_no_row_of_integers_are_refused(bad, side):
    bq = BlockQuantizer(40, context=NoContext())
    c = codes(4, 40)
    good = [0] * (len(bad) - 1) + [4] if np.ndim(bad) else [0, 4]
    args = [bad, good] if side == 0 else [good, bad]
    with pytest.raises(Configuration) as e:
        bq.grouped_product(c, args[0], c, args[1], out_size=16)
    assert e.value.parameter == "offsets"

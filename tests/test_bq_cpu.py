"""The block quantiser's refusals that need no device: arguments that the host mirror checks, and null handles."""
import ctypes as C

import numpy as np
import pytest

from proxima_b200 import _native as N
from proxima_b200.blockquant import BlockCodes, BlockQuantizer
from proxima_b200.errors import Configuration, DimensionMismatch


class NoContext:
    """Stands for a context: nothing here reaches the device."""

    handle = None
    device = 0


def codes(n, dim, ld=None, sld=None):
    blocks = -(-dim // 128)
    return BlockCodes(np.zeros((n, ld or -(-dim // 16) * 16), np.uint8),
                      np.zeros((n, sld or -(-blocks // 4) * 4), np.uint8), dim)


@pytest.fixture
def bq():
    return BlockQuantizer(40, context=NoContext())


@pytest.mark.parametrize("dim", [0, -3, (1 << 20) + 1])
def test_dimension_is_refused(dim):
    with pytest.raises(Configuration) as e:
        BlockQuantizer(dim, context=NoContext())
    assert e.value.parameter == "dim"


def test_shapes_and_types_are_refused(bq):
    good = codes(5, 40)
    with pytest.raises(DimensionMismatch):
        bq.encode(np.zeros((3, 41), np.float32))
    with pytest.raises(DimensionMismatch):
        bq.encode(np.zeros((2, 3, 40), np.float32))
    with pytest.raises(DimensionMismatch):
        bq.decode(codes(5, 48))
    with pytest.raises(Configuration):  # pitch below the dimension rounded up
        bq.decode(BlockCodes(good.codes[:, :32], good.scales, 40))
    with pytest.raises(Configuration):  # pitch not a multiple of 16
        bq.decode(codes(5, 40, ld=56))
    with pytest.raises(Configuration):  # components not contiguous
        bq.decode(BlockCodes(np.zeros((5, 96), np.uint8)[:, ::2], good.scales, 40))
    with pytest.raises(Configuration):
        bq.decode(BlockCodes(good.codes.astype(np.int16), good.scales, 40))
    with pytest.raises(Configuration):  # rows of codes and scales differ in number
        bq.product(BlockCodes(good.codes, good.scales[:3], 40), good)
    with pytest.raises(Configuration) as e:
        bq.decode(good, dtype=np.float64)
    assert e.value.parameter == "dtype"
    with pytest.raises(Configuration):
        bq.product(good, good, dtype=np.int8)
    with pytest.raises(Configuration):
        bq.product(good, good, out=np.zeros((5, 5), np.float32))
    with pytest.raises(TypeError):
        good[2]


def test_group_arguments_are_refused(bq):
    q, b = codes(5, 40), codes(7, 40)
    with pytest.raises(Configuration):  # 7 rows over 2 groups without offsets
        bq.grouped_product(q, [0, 2, 5], b)
    with pytest.raises(Configuration):
        bq.grouped_product(q, [0], b)
    with pytest.raises(Configuration):
        bq.grouped_product(q, None, b)
    with pytest.raises(Configuration):  # lengths differ
        bq.grouped_product(q, [0, 2, 5], b, [0, 7])
    with pytest.raises(Configuration):  # falling
        bq.grouped_product(q, [0, 5, 0], b, [0, 0, 7])


def test_row_slices_are_views():
    c = codes(9, 200)
    part = c[2:5]
    assert len(part) == 3 and part.dim == 200 and part.codes.base is c.codes
    assert c.bytes_per_vector == 208 + 4


def test_null_context_is_a_status_and_no_crash():
    lib = N.load()
    rows = N.PxcBqRows(None, None, 0, 16, 4)
    err = N.PxcError()
    for status in (
        lib.pxc_bq_encode(None, None, 0, 8, 8, C.byref(rows), C.byref(err)),
        lib.pxc_bq_encode_device(None, None, 0, 8, 8, C.byref(rows), None, C.byref(err)),
        lib.pxc_bq_decode(None, C.byref(rows), 8, None, 0, 8, C.byref(err)),
        lib.pxc_bq_decode_device(None, C.byref(rows), 8, None, 0, 8, None, C.byref(err)),
        lib.pxc_bq_product(None, C.byref(rows), C.byref(rows), 8, None, 0, 8, C.byref(err)),
        lib.pxc_bq_product_device(None, C.byref(rows), C.byref(rows), 8, None, 0, 8, None, C.byref(err)),
        lib.pxc_bq_grouped_product(None, C.byref(rows), None, C.byref(rows), None, 1, 8, None, 0, 0, C.byref(err)),
        lib.pxc_bq_grouped_product_device(None, C.byref(rows), None, C.byref(rows), None, 1, 8, None, 0, 0, None,
                                          C.byref(err)),
        lib.pxc_bq_check(None, None, C.byref(err)),
    ):
        assert status == 7 and err.parameter == b"ctx"
        assert lib.pxc_bq_check(None, None, None) == 7  # no error struct

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


def test_null_contexts_are_a_status_and_no_crash():
    lib = N.load()
    rows = N.PxcBqRows(None, None, 0, 16, 4)
    err = N.PxcError()
    r, e = C.byref(rows), C.byref(err)
    for status in (
        lib.pxc_bq_encode_as(None, 7, None, 0, 8, 8, r, None, e),
        lib.pxc_bq_decode_as(None, 7, r, 8, None, 0, 8, None, e),
        lib.pxc_bq_product_as(None, 7, r, r, 8, None, 0, 8, None, e),
        lib.pxc_bq_grouped_product_as(None, 7, r, None, r, None, 1, 8, None, 0, 0, None, e),
        lib.pxc_bq_report_as(None, 7, e),
        lib.pxc_bq_check_as(None, 7, None, e),
        lib.pxc_bq_forget(None, None, 0, e),
    ):
        assert status == 7 and err.parameter == b"ctx"


def test_callers_numbers_are_given_out_once():
    lib = N.load()
    a, b, c = lib.pxc_bq_callers(5), lib.pxc_bq_callers(1), lib.pxc_bq_callers(1)
    assert a > 0 and b == a + 5 and c == b + 1
    own = [BlockQuantizer(40, context=NoContext())._caller for _ in range(100)]
    assert len(set(own)) == 100


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


class OnDevice:
    """Stands for a CUDA tensor."""

    is_cuda = True
    ndim = 2


def test_host_tensors_are_taken_or_refused_like_arrays():
    torch = pytest.importorskip("torch")
    bq = BlockQuantizer(40, context=NoContext())
    c = codes(4, 40)
    t = BlockCodes(torch.from_numpy(c.codes), torch.from_numpy(c.scales), 40)
    a, b = bq._rows(c, False, "c"), bq._rows(t, False, "t")
    assert [getattr(a, f) for f, _ in N.PxcBqRows._fields_] == [getattr(b, f) for f, _ in N.PxcBqRows._fields_]
    for bad in (BlockCodes(t.codes.view(torch.float8_e4m3fn), t.scales, 40), BlockCodes(t.codes.long(), t.scales, 40),
                BlockCodes(t.codes, c.scales.tolist(), 40), BlockCodes(t.codes, OnDevice(), 40),
                BlockCodes(t.codes.t(), t.scales, 40), BlockCodes(t.codes[:, ::2], t.scales, 40)):
        with pytest.raises(Configuration) as e:
            bq.decode(bad)
        assert e.value.parameter == "codes"
        with pytest.raises(Configuration) as e:
            bq.product(t, bad)
        assert e.value.parameter == "base"
    with pytest.raises(Configuration) as e:
        bq.grouped_product(c, OnDevice(), c)
    assert e.value.parameter == "offsets"


def test_host_vectors_of_any_tensor():
    torch = pytest.importorskip("torch")
    bq = BlockQuantizer(40, context=NoContext())
    x = torch.randn((3, 40), generator=torch.Generator().manual_seed(1))
    for v in (x, x.half(), x.bfloat16(), x.clone().requires_grad_()):
        got = bq._vectors(v)
        assert got.dtype == (np.float16 if v.dtype == torch.float16 else np.float32)
        assert np.array_equal(got, v.detach().float().numpy())


@pytest.mark.parametrize("dtype", [">f4", ">f2", np.dtype(np.float16).newbyteorder()])
def test_results_in_another_byte_order_are_refused(dtype):
    bq = BlockQuantizer(40, context=NoContext())
    c = codes(4, 40)
    for call in (lambda: bq.decode(c, dtype=dtype), lambda: bq.product(c, c, dtype=dtype),
                 lambda: bq.grouped_product(c, [0, 4], c, dtype=dtype)):
        with pytest.raises(Configuration) as e:
            call()
        assert e.value.parameter == "dtype"

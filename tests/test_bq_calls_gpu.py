"""Ways of calling the block quantiser that the documentation allows."""
import ctypes as C
import threading

import numpy as np
import pytest

from proxima_b200 import _native as N
from proxima_b200.blockquant import BlockCodes, BlockQuantizer
from proxima_b200.errors import Configuration, Internal

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def codes_of(bq, rows, seed):
    """Small integers: products of them are exact in any order."""
    g = torch.Generator().manual_seed(seed)
    return bq.encode(torch.randint(-3, 4, (rows, bq.dim), generator=g).float().cuda())


def in_a_thread(call):
    """What `call` returns in a thread that has made no CUDA call before."""
    got = []

    def work():
        try:
            got.append(call())
        except BaseException as e:
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(got[0], BaseException):
        raise got[0]
    return got[0]


def test_a_products_thread_needs_no_cuda_call_before():
    bq = BlockQuantizer(48)
    q, b = codes_of(bq, 20, 1), codes_of(bq, 40, 2)
    off = torch.tensor([0, 7, 20], device="cuda")
    want, parts = bq.product(q, b), bq.grouped_product(q, off, b)
    out = torch.empty((20, 40), device="cuda")
    torch.cuda.synchronize()
    in_a_thread(lambda: bq.product(q, b, out=out))
    assert torch.equal(out, want)
    assert torch.equal(in_a_thread(lambda: bq.product(q, b)), want)
    assert torch.equal(in_a_thread(lambda: bq.grouped_product(q, off, b)), parts)
    assert torch.equal(in_a_thread(lambda: bq.encode(bq.decode(q))).codes, q.codes)
    h = BlockCodes(q.codes.cpu().numpy(), q.scales.cpu().numpy(), 48)
    assert np.array_equal(in_a_thread(lambda: bq.product(h, h)), bq.product(q, q).cpu().numpy())


def test_a_call_after_one_that_found_no_memory():
    """300,000 x 300,000 scores are 360 GB, more than the device has; the next call has nothing to do with it."""
    bq = BlockQuantizer(16)
    x = torch.ones((3, 16), device="cuda")
    want = bq.encode(x)
    h = BlockCodes(np.zeros((300_000, 16), np.uint8), np.zeros((300_000, 4), np.uint8), 16)
    rows, out = bq._rows(h, False, "h"), np.zeros(16, np.float32)
    with pytest.raises(Internal):
        N.call("pxc_bq_product", bq.ctx.handle, C.byref(rows), C.byref(rows), 16, out.ctypes.data, 0, 300_000)
    got = bq.encode(x)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


def test_host_tensors_give_the_arrays_results():
    bq = BlockQuantizer(150)
    x = torch.randn((30, 150), generator=torch.Generator().manual_seed(1))
    for v in (x, x.half(), x.bfloat16(), x.clone().requires_grad_()):
        got, want = bq.encode(v), bq.encode(v.detach().cuda())
        assert isinstance(got.codes, np.ndarray)
        assert np.array_equal(got.codes, want.codes.cpu().numpy()) and np.array_equal(got.scales, want.scales.cpu().numpy())
    t = BlockCodes(torch.from_numpy(got.codes), torch.from_numpy(got.scales), 150)
    assert np.array_equal(bq.decode(t), bq.decode(got))
    assert np.array_equal(bq.product(t[3:9], t), bq.product(got[3:9], got))
    off = torch.tensor([0, 9, 30])
    assert np.array_equal(bq.grouped_product(t, off, t, off), bq.grouped_product(got, off.numpy(), got, off.numpy()))

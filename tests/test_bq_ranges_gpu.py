"""The block quantiser at the ends of its ranges: scales, magnitudes, dimensions, sizes, pitches."""
import ctypes as C
import threading

import numpy as np
import pytest

from proxima_b200 import _native as N
from proxima_b200.blockquant import BlockCodes, BlockQuantizer

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def whole_codes(rows, dim, seed):
    """Rows of whole numbers up to 3 under scales of 1, and their values."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-3, 4, (rows, dim), generator=g, device="cuda").float()
    ld, blocks = -(-dim // 16) * 16, -(-dim // 128)
    codes = torch.zeros((rows, ld), dtype=torch.uint8, device="cuda")
    codes[:, :dim] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device="cuda")
    return BlockCodes(codes, scales, dim), v


# ---- what a sum keeps ----
@pytest.mark.parametrize("ones", [1, 2, 16])
def test_every_pair_of_scale_bytes(ones):
    """Powers of two as products: exact from the least value below the normal range to the largest, infinite above."""
    codes = torch.zeros((255, 16), dtype=torch.uint8, device="cuda")
    codes[:, :ones] = 0x38  # 1.0
    scales = torch.zeros((255, 4), dtype=torch.uint8, device="cuda")
    scales[:, 0] = torch.arange(255, device="cuda").to(torch.uint8)
    c = BlockCodes(codes, scales, 16)
    got = BlockQuantizer(16).product(c, c).double().cpu().numpy()
    e = np.arange(255)[:, None] + np.arange(255)[None, :] - 254 + int(np.log2(ones))
    want = np.where(e > 127, np.inf, np.exp2(np.minimum(e, 127).astype(np.float64)))
    held = e >= -149
    assert np.array_equal(got[held], want[held])
    # 2**-150 lies half way to the least value and goes to the even one, 0, like all below
    assert not got[~held].any()


@pytest.mark.parametrize("dim", [64, 128, 160, 2048, 8192])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_small_terms_beside_a_large_sum(dim, where):
    """One product of 2**22 and whole numbers up to 9 beside it: every partial sum in any order is a whole number below
    2**24, so a sum that keeps 24 bits is exact, the terms added in one step with the large one among them."""
    q, qv = whole_codes(40, dim, 1)
    b, bv = whole_codes(300, dim, 2)
    at = {"first": 0, "middle": dim // 2, "last": dim - 1}[where]
    if dim <= 128:  # beside the others of its block: 256 under a scale of 8, the others eighths
        q.scales[:, 0], b.scales[:, 0] = 127 + 3, 127 + 3
        q.codes[:, :dim] = (qv / 8).to(torch.float8_e4m3fn).view(torch.uint8)
        b.codes[:, :dim] = (bv / 8).to(torch.float8_e4m3fn).view(torch.uint8)
        large = torch.full((1,), 256.0).to(torch.float8_e4m3fn).view(torch.uint8).item()  # 2**11 once scaled
        q.codes[:, at], b.codes[:, at] = large, large
        qv[:, at], bv[:, at] = 2048, 2048
    else:  # alone in its block
        block = at // 128 * 128
        q.codes[:, block:block + 128], b.codes[:, block:block + 128] = 0, 0
        qv[:, block:block + 128], bv[:, block:block + 128] = 0, 0
        q.scales[:, at // 128], b.scales[:, at // 128] = 127 + 11, 127 + 11
        q.codes[:, at], b.codes[:, at] = 0x38, 0x38
        qv[:, at], bv[:, at] = 2048, 2048
    want = qv.double() @ bv.double().t()
    assert want.abs().max() < 2**24
    assert torch.equal(BlockQuantizer(dim).product(q, b).double(), want)


@pytest.mark.parametrize("nq,n,dim", [(30, 200, 4096), (300, 300, 16_384), (5, 700, 65_536), (230, 130, 100_003),
                                       (3, 130, 1 << 20), (240, 300, 1 << 20)])
def test_long_sums_of_whole_numbers_are_exact(nq, n, dim):
    """|partial sums| <= 9 * dim < 2**24."""
    q, qv = whole_codes(nq, dim, 3)
    b, bv = whole_codes(n, dim, 4)
    got = BlockQuantizer(dim).product(q, b)
    want = torch.zeros((nq, n), dtype=torch.float64, device="cuda")
    for i in range(0, dim, 1 << 16):
        want += qv[:, i:i + (1 << 16)].double() @ bv[:, i:i + (1 << 16)].double().t()
    assert torch.equal(got.double(), want)


# ---- sizes past 31 and 32 bits ----
def test_an_output_of_more_than_2_31_values():
    nq, n, dim = 70_001, 40_003, 16  # 2.8e9 values, 5.6 GB
    q, qv = whole_codes(nq, dim, 5)
    b, bv = whole_codes(n, dim, 6)
    got = BlockQuantizer(dim).product(q, b, dtype=torch.bfloat16)  # up to 144: exact in 8 bits
    for i in range(0, nq, 7001):
        want = (qv[i:i + 7001] @ bv.t()).to(torch.bfloat16)
        assert torch.equal(got[i:i + 7001], want)


def test_groups_whose_matrices_pass_2_31_values():
    dim = 16
    qo, bo = np.array([0, 60_000, 60_000, 80_001]), np.array([0, 31_000, 31_001, 51_002])
    size = 60_000 * 31_000 + 20_001 * 20_001  # 2.26e9
    q, qv = whole_codes(80_001, dim, 7)
    b, bv = whole_codes(51_002, dim, 8)
    got = BlockQuantizer(dim).grouped_product(q, torch.from_numpy(qo).cuda(), b, torch.from_numpy(bo).cuda(), out_size=size,
                                              dtype=torch.bfloat16)
    first = got[:60_000 * 31_000].view(60_000, 31_000)
    for i in range(0, 60_000, 6000):
        assert torch.equal(first[i:i + 6000], (qv[i:i + 6000] @ bv[:31_000].t()).to(torch.bfloat16))
    last = got[60_000 * 31_000:].view(20_001, 20_001)
    for i in range(0, 20_001, 5000):
        assert torch.equal(last[i:i + 5000], (qv[60_000 + i:60_000 + i + 5000] @ bv[31_001:].t())[:20_001].to(torch.bfloat16))


@pytest.mark.parametrize("n,dim", [(150_000_001, 16), (4_500_003, 500)])
def test_codes_of_more_than_2_31_components(n, dim):
    g = torch.Generator(device="cuda").manual_seed(9)
    few = torch.randn((1000, dim), generator=g, device="cuda").half()
    x = torch.empty((n, dim), dtype=torch.float16, device="cuda")
    x[:n // 1000 * 1000].view(-1, 1000, dim).copy_(few)
    x[n // 1000 * 1000:] = few[:n % 1000]
    bq = BlockQuantizer(dim)
    small = bq.encode(few)
    want = bq.decode(small, dtype=torch.float16)
    c = bq.encode(x)
    ld, sld, whole = c.codes.shape[1], c.scales.shape[1], n // 1000 * 1000
    assert (c.codes[:whole].view(-1, 1000, ld) == small.codes).all() and torch.equal(c.codes[whole:], small.codes[:n % 1000])
    assert (c.scales[:whole].view(-1, 1000, sld) == small.scales).all()
    del x
    back = bq.decode(c, dtype=torch.float16)
    assert (back[:whole].view(-1, 1000, dim) == want).all() and torch.equal(back[whole:], want[:n % 1000])


# ---- pitches ----
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,stride,offset", [(128, 129, 0), (96, 97, 1), (300, 304, 0), (300, 303, 2), (1001, 1003, 5),
                                               (64, 64, 1), (31, 31, 3), (31, 40, 0), (1, 7, 2), (257, 257, 0)])
def test_decode_into_strided_and_unaligned_rows(dim, stride, offset, kind):
    rows, dtype = 37, DTYPES[kind]
    bq = BlockQuantizer(dim)
    c = bq.encode(torch.randn((rows, dim), generator=torch.Generator().manual_seed(dim)).cuda())
    want = bq.decode(c, dtype=dtype)
    flat = torch.full((offset + rows * stride + 64,), -7.0, dtype=dtype, device="cuda")
    out = torch.as_strided(flat, (rows, dim), (stride, 1), offset)
    r = bq._rows(c, True, "c")
    N.call("pxc_bq_decode_device", bq.ctx.handle, C.byref(r), dim, out.data_ptr(), ["f32", "f16", "bf16"].index(kind), stride, 1)
    expect = torch.full_like(flat, -7.0)
    torch.as_strided(expect, (rows, dim), (stride, 1), offset).copy_(want)
    assert torch.equal(flat, expect)


@pytest.mark.parametrize("dim,pad", [(768, 0), (333, 0), (96, 37)])
def test_host_rows_of_any_size_and_pitch(dim, pad):
    """Host forms through the C functions: pitches of vectors, codes, scales and results wider than the rows."""
    nq, n = 64, 20_000
    g = np.random.default_rng(10)
    bq = BlockQuantizer(dim)
    x = g.standard_normal((n, dim + pad)).astype(np.float32)
    y = g.standard_normal((nq, dim)).astype(np.float32)
    dx, dy = bq.encode(torch.from_numpy(x[:, :dim].copy()).cuda()), bq.encode(torch.from_numpy(y).cuda())
    ld, sld = -(-dim // 16) * 16 + 16 * (pad > 0), -(-bq.blocks // 4) * 4 + 4 * (pad > 0)
    codes, scales = np.full((n, ld), 0xAB, np.uint8), np.full((n, sld), 0xCD, np.uint8)
    rows = N.PxcBqRows(codes.ctypes.data, scales.ctypes.data, n, ld, sld)
    N.call("pxc_bq_encode", bq.ctx.handle, x.ctypes.data, 0, dim + pad, dim, C.byref(rows))
    w, sw = dx.codes.shape[1], dx.scales.shape[1]
    assert np.array_equal(codes[:, :w], dx.codes.cpu().numpy()) and (codes[:, w:] == 0xAB).all()
    assert np.array_equal(scales[:, :sw], dx.scales.cpu().numpy()) and (scales[:, sw:] == 0xCD).all()
    out = np.full((n, dim + pad), -7.0, np.float32)
    N.call("pxc_bq_decode", bq.ctx.handle, C.byref(rows), dim, out.ctypes.data, 0, dim + pad)
    assert np.array_equal(out[:, :dim], bq.decode(dx).cpu().numpy()) and (out[:, dim:] == -7).all()
    q = bq.encode(y)
    qr = bq._rows(q, False, "q")
    scores = np.full((nq, n + pad), -7.0, np.float32)
    N.call("pxc_bq_product", bq.ctx.handle, C.byref(qr), C.byref(rows), dim, scores.ctypes.data, 0, n + pad)
    assert np.array_equal(scores[:, :n], bq.product(dy, dx).cpu().numpy()) and (scores[:, n:] == -7).all()


# ---- beside one another ----
def test_every_result_of_several_streams_and_threads():
    dim, rounds = 500, 20
    q, qv = whole_codes(150, dim, 11)
    b, bv = whole_codes(2000, dim, 12)
    want = qv @ bv.t()
    bq = BlockQuantizer(dim)
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                mine = [bq.product(q, b) for _ in range(rounds)]
                torch.cuda.current_stream().synchronize()
            results[i] = mine
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(results) == 3
    assert all(len(r) == rounds and all(torch.equal(x, want) for x in r) for r in results.values())


def test_the_first_calls_of_a_context_may_be_captured():
    from proxima_b200.index import Context

    ctx = Context(0)
    bq = BlockQuantizer(192, context=ctx)
    x = torch.randn((60, 192), generator=torch.Generator().manual_seed(13)).cuda()
    off = torch.tensor([0, 60], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = bq.encode(x)
        full, back = bq.product(c, c), bq.decode(c)
        flat = bq.grouped_product(c, off, c, off, out_size=3600)
    for seed in (14, 15):
        x.copy_(torch.randn((60, 192), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        own = BlockQuantizer(192)
        d = own.encode(x)
        assert torch.equal(full, own.product(d, d)) and torch.equal(back, own.decode(d))
        assert torch.equal(flat.view(60, 60), full)
    bq.check()
    del graph
    ctx.close()


# ---- groups of many queries ----
@pytest.mark.parametrize("mq,mb,dim", [
    ([900], [600], 200),
    ([600, 512, 700], [513, 600, 900], 130),
    ([3000, 0, 5, 1], [200, 3000, 1, 77], 96),  # one group holds nearly all
    ([800] * 7, [128] * 7, 64),  # no more rows than one CTA takes
    ([4000, 1, 600, 0, 17], [1, 1700, 0, 128, 900], 520),
    ([256] * 9, [300] * 9, 256),
    ([513] * 4, [516] * 4, 300),
])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_groups_of_many_queries_are_exact(mq, mb, dim, kind):
    qo, bo = np.concatenate([[0], np.cumsum(mq)]), np.concatenate([[0], np.cumsum(mb)])
    q, qv = whole_codes(int(qo[-1]), dim, 16)
    b, bv = whole_codes(int(bo[-1]), dim, 17)
    parts = [qv[qo[g]:qo[g + 1]] @ bv[bo[g]:bo[g + 1]].t() for g in range(len(mq))]
    want = torch.cat([p.reshape(-1) for p in parts]).to(DTYPES[kind])
    tq, tb = torch.from_numpy(qo).cuda(), torch.from_numpy(bo).cuda()
    got = BlockQuantizer(dim).grouped_product(q, tq, b, tb, out_size=len(want), dtype=DTYPES[kind])
    assert torch.equal(got, want)
    if len(set(mb)) == 1:
        even = BlockQuantizer(dim).grouped_product(q, tq, b, dtype=DTYPES[kind])
        assert torch.equal(even.reshape(-1), want)

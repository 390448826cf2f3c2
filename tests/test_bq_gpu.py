"""The block quantiser on the GPU against plain 64-bit computations.

Encoding and decoding are exact rules, compared bit for bit. Products are compared in two ways:
inputs whose sums every order gets exactly (small integers with power-of-two scales), bit for
bit, and random inputs within the bound of 32-bit sums. For those the tensor core adds
groups of 32 products to the sum, each term cut to 24 bits or more of the largest: at most 33
errors of 2**-23 of the sum of magnitudes per group, so (dim + 64) * 2**-23 * sum |q_i b_i| in
all; the output's rounding adds half a step.
"""
import ctypes as C

import numpy as np
import pytest

from proxima_b200 import _native as N
from proxima_b200.blockquant import BlockCodes, BlockQuantizer
from proxima_b200.errors import Configuration, ProximaError

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the definition in 64 bits ----
def e4m3_round(u):
    """|u| <= 448 to the e4m3 grid, nearest, ties to even."""
    with np.errstate(invalid="ignore"):
        _, e = np.frexp(np.abs(u))
        step = np.exp2(np.maximum(e - 1.0, -6.0) - 3.0)
        return np.round(u / step) * step


def encode_ref(x):
    """(values on the grid, exponents) of rows in 64 bits."""
    x = np.asarray(x, np.float64)
    n, dim = x.shape
    blocks = -(-dim // 128)
    p = np.zeros((n, blocks * 128))
    p[:, :dim] = x
    p = p.reshape(n, blocks, 128)
    top = np.where(np.isfinite(p), np.abs(p), 0).max(2)
    m, e = np.frexp(top)
    s = np.where(m <= 0.875, e - 9, e - 8)
    s = np.maximum(np.where(top == 0, 0, s), -126)
    u = np.clip(p / np.exp2(s.astype(np.float64))[:, :, None], -448, 448)
    return e4m3_round(u), s


def rows_ref(grid, s, dim):
    return (grid * np.exp2(s.astype(np.float64))[:, :, None]).reshape(len(grid), -1)[:, :dim]


def code_values(c):
    """What BlockCodes (tensors) hold, in 64 bits."""
    grid = c.codes[:, :c.dim].view(torch.float8_e4m3fn).double().cpu().numpy()
    blocks = -(-c.dim // 128)
    s = np.exp2(c.scales[:, :blocks].double().cpu().numpy() - 127.0)
    return grid * np.repeat(s, 128, axis=1)[:, :c.dim]


def bound(q, b, dtype):
    """(reference, tolerance) of the product of two 64-bit matrices."""
    ref = q @ b.T
    return ref, tolerance(ref, np.abs(q) @ np.abs(b).T, q.shape[1], dtype)


def tolerance(ref, magnitudes, dim, dtype):
    tol = (dim + 64) * 2.0**-23 * magnitudes
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(ref) + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return tol


def exact_codes(n, dim, seed):
    """Rows with codes from {-3..3} and block scales 2**-2..2**2: every product sum is a multiple
    of 2**-4 below 2**16 * 9 * dim / 2**16, so 32-bit sums in any order are exact for dim <= 2**12."""
    g = np.random.default_rng(seed)
    blocks = -(-dim // 128)
    v = g.integers(-3, 4, (n, dim)).astype(np.float32)
    s = g.integers(-2, 3, (n, blocks))
    ld, sld = -(-dim // 16) * 16, -(-blocks // 4) * 4
    codes = torch.zeros((n, ld), dtype=torch.uint8)
    codes[:, :dim] = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8)
    # the pitch beyond the dimension holds NaN codes: nothing may read them into a sum
    codes[:, dim:] = 0x7F
    scales = torch.full((n, sld), 255, dtype=torch.uint8)
    scales[:, :blocks] = torch.from_numpy((s + 127).astype(np.uint8))
    values = v.astype(np.float64) * np.repeat(np.exp2(s.astype(np.float64)), 128, axis=1)[:, :dim]
    return BlockCodes(codes.cuda(), scales.cuda(), dim), values


# ---- codes ----
def special_rows(dim, seed, dtype):
    """Ordinary rows, then rows at the rule's edges."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((24, dim), generator=g) * torch.exp(2 * torch.randn((24, 1), generator=g))
    f = torch.finfo(dtype)
    x[1] = 0.0
    x[2] = -0.0
    x[3] = f.max  # the largest scale of the type
    x[4] = f.tiny * 3  # the smallest normals
    x[5] = f.smallest_normal * f.eps  # the least subnormal
    x[6] = 448.0
    x[7] = 449.0  # one step up in scale
    x[8, ::2] = 448.0
    x[8, 1::2] = 17.0  # 17 and 19 lie half way between two codes
    x[9, ::2] = 448.0
    x[9, 1::2] = 19.0
    x[10, ::3] = float("inf")
    x[11, ::3] = -float("inf")
    x[12, 0] = float("nan")
    x[13] = float("inf")
    x[14] = float("nan")
    x[15, :] = 2.0**-9 * 1.5  # below the first code once a large one sits beside it
    x[15, -1] = 448.0
    x[16] = torch.linspace(-1, 1, dim)
    return x.to(dtype)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [1, 7, 9, 15, 16, 17, 31, 96, 127, 128, 129, 131, 250, 257, 300, 768, 1001, 4096])
def test_encode_and_decode_are_the_definition(dim, kind):
    dtype = DTYPES[kind]
    x = special_rows(dim, dim, dtype)
    bq = BlockQuantizer(dim)
    c = bq.encode(x.cuda())
    grid, s = encode_ref(x.double().numpy())
    blocks = bq.blocks
    scales = c.scales.cpu().numpy().astype(int)
    assert np.array_equal(scales[:, :blocks] - 127, s)
    assert not scales[:, blocks:].any()
    got = c.codes[:, :dim].view(torch.float8_e4m3fn).double().cpu().numpy()
    assert np.array_equal(got, grid.reshape(len(x), -1)[:, :dim], equal_nan=True)
    assert not c.codes[:, dim:].cpu().numpy().any()
    for out in DTYPES.values():
        want = torch.from_numpy(rows_ref(grid, s, dim)).to(torch.float32).to(out)
        back = bq.decode(c, dtype=out).cpu()
        assert torch.equal(torch.nan_to_num(back, nan=-7.0), torch.nan_to_num(want, nan=-7.0))
    assert torch.equal(torch.signbit(bq.decode(c).cpu()[2]), torch.ones(dim, dtype=torch.bool))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,pitch,offset", [(96, 97, 0), (128, 128, 1), (300, 304, 4), (130, 136, 8), (64, 200, 3)])
def test_encode_reads_strided_and_unaligned_rows(dim, pitch, offset, kind):
    flat = torch.randn(20 * pitch + offset + dim, generator=torch.Generator().manual_seed(1)).to(DTYPES[kind]).cuda()
    x = torch.as_strided(flat, (20, dim), (pitch, 1), offset)
    bq = BlockQuantizer(dim)
    a, b = bq.encode(x), bq.encode(x.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    t = torch.randn((dim, 9), generator=torch.Generator().manual_seed(2)).to(DTYPES[kind]).cuda()
    c, d = bq.encode(t.t()), bq.encode(t.t().contiguous())  # columns: copied first
    assert torch.equal(c.codes, d.codes) and torch.equal(c.scales, d.scales)


@pytest.mark.parametrize("rows", [1, 3, 1000])
def test_pitches_wider_than_needed_are_left_alone(rows):
    dim, ld, sld = 200, 256, 12
    x = torch.randn((rows, dim), generator=torch.Generator().manual_seed(3)).cuda()
    bq = BlockQuantizer(dim)
    codes = torch.full((rows, ld), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows, sld), 0xCD, dtype=torch.uint8, device="cuda")
    r = N.PxcBqRows(codes.data_ptr(), scales.data_ptr(), rows, ld, sld)
    N.call("pxc_bq_encode_device", bq.ctx.handle, x.data_ptr(), 0, dim, dim, C.byref(r), 1)
    torch.cuda.synchronize()
    want = bq.encode(x)
    assert torch.equal(codes[:, :208], want.codes) and torch.equal(scales[:, :4], want.scales)
    assert (codes[:, 208:] == 0xAB).all() and (scales[:, 4:] == 0xCD).all()
    out = torch.full((rows, 260), -1.0, device="cuda")
    N.call("pxc_bq_decode_device", bq.ctx.handle, C.byref(r), dim, out.data_ptr(), 0, 260, 1)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :dim], bq.decode(want)) and (out[:, dim:] == -1).all()


def test_decode_takes_any_scale_byte():
    codes = torch.full((256, 16), 0x38, dtype=torch.uint8, device="cuda")  # 1.0
    scales = torch.zeros((256, 4), dtype=torch.uint8, device="cuda")
    scales[:, 0] = torch.arange(256, device="cuda").to(torch.uint8)
    got = BlockQuantizer(16).decode(BlockCodes(codes, scales, 16)).double().cpu().numpy()[:, 0]
    assert np.array_equal(got[:255], np.exp2(np.arange(255) - 127.0)) and np.isnan(got[255])


# ---- products ----
SHAPES = [(1, 1, 1), (1, 127, 128), (1, 1000, 96), (3, 129, 64), (16, 128, 128), (17, 300, 130), (64, 64, 512),
          (65, 200, 513), (200, 333, 260), (223, 130, 640), (224, 128, 128), (225, 131, 1100), (257, 512, 768),
          (500, 77, 2048), (700, 1111, 384), (2, 40000, 16), (4000, 5, 200), (700, 17000, 48),
          # few queries over so many rows that a tile takes several times 128 of them
          (1, 75776, 129), (3, 75000, 40), (40, 75700, 513), (60, 37800, 130)]


@pytest.mark.parametrize("nq,n,dim", SHAPES)
def test_product_of_exact_inputs_is_exact(nq, n, dim):
    q, qv = exact_codes(nq, dim, 1)
    b, bv = exact_codes(n, dim, 2)
    got = BlockQuantizer(dim).product(q, b)
    assert np.array_equal(got.double().cpu().numpy(), qv @ bv.T)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,n,dim", [(1, 4099, 768), (5, 700, 100), (130, 257, 1000), (300, 600, 4096), (37, 1003, 96)])
def test_product_within_the_bound_of_its_sums(nq, n, dim, kind):
    g = torch.Generator().manual_seed(nq)
    bq = BlockQuantizer(dim)
    q = bq.encode((torch.randn((nq, dim), generator=g) * torch.exp(torch.randn(dim, generator=g))).cuda())
    b = bq.encode(torch.randn((n, dim), generator=g).cuda())
    out = DTYPES[kind]
    got = bq.product(q, b, dtype=out)
    assert got.dtype == out
    ref, tol = bound(code_values(q), code_values(b), out)
    assert (np.abs(got.double().cpu().numpy() - ref) <= tol).all()


def test_product_writes_only_its_rows_and_reads_slices():
    dim = 150
    q, qv = exact_codes(40, dim, 3)
    b, bv = exact_codes(300, dim, 4)
    out = torch.full((50, 320), -5.0, device="cuda")
    bq = BlockQuantizer(dim)
    got = bq.product(q[7:30], b[11:290], out=out[3:26, 1:280])
    assert got.data_ptr() == out[3:26, 1:280].data_ptr()
    want = np.full((50, 320), -5.0)
    want[3:26, 1:280] = qv[7:30] @ bv[11:290].T
    assert np.array_equal(out.double().cpu().numpy(), want)


@pytest.mark.parametrize("nq,n", [(0, 5), (5, 0), (0, 0)])
def test_products_of_nothing(nq, n):
    bq = BlockQuantizer(24)
    q, b = bq.encode(torch.zeros((nq, 24), device="cuda")), bq.encode(torch.zeros((n, 24), device="cuda"))
    assert bq.product(q, b).shape == (nq, n)
    off = torch.tensor([0, nq], device="cuda")
    assert bq.grouped_product(q, off, b).shape == (nq, n)
    assert bq.grouped_product(q, off, b, torch.tensor([0, n], device="cuda")).shape == (0,)
    assert bq.decode(q).shape == (nq, 24)


def test_a_nan_stays_in_its_row_and_column():
    dim = 260
    q, qv = exact_codes(30, dim, 5)
    b, bv = exact_codes(200, dim, 6)
    q.codes[4, 259] = 0x7F
    b.scales[9, 1] = 255
    got = BlockQuantizer(dim).product(q, b).double().cpu().numpy()
    assert np.isnan(got[4]).all() and np.isnan(got[:, 9]).all()
    want = qv @ bv.T
    rows, cols = np.arange(30) != 4, np.arange(200) != 9
    assert np.array_equal(got[np.ix_(rows, cols)], want[np.ix_(rows, cols)])


def test_scales_far_apart():
    """Blocks whose scales differ by 2**40 and pairs whose product leaves 32 bits."""
    dim = 256
    x = torch.ones((6, dim))
    for i, e in enumerate((-100, -60, -20, 20, 60, 100)):
        x[i, :128] = 2.0**e
        x[i, 128:] = 2.0 ** (e - 20)
    bq = BlockQuantizer(dim)
    c = bq.encode(x.cuda())
    v = code_values(c)
    assert np.array_equal(v, x.double().numpy())
    ref = v @ v.T
    got = bq.product(c, c).double().cpu().numpy()
    big = np.abs(ref) > torch.finfo(torch.float32).max
    small = np.abs(ref) < 2.0**-100
    assert np.isposinf(got[big]).all() and (got[small] >= 0).all() and (got[small] < 2.0**-99).all()
    mid = ~big & ~small
    assert mid.sum() >= 16 and (np.abs(got[mid] - ref[mid]) <= 2.0**-20 * ref[mid]).all()


def test_products_take_any_scale_byte():
    """Every pair of bytes whose product of powers stays within 32 bits, the two ends among them."""
    codes = torch.full((255, 16), 0x38, dtype=torch.uint8, device="cuda")  # 1.0
    scales = torch.zeros((255, 4), dtype=torch.uint8, device="cuda")
    scales[:, 0] = torch.arange(255, device="cuda").to(torch.uint8)
    c = BlockCodes(codes, scales, 16)
    got = BlockQuantizer(16).product(c, c).double().cpu().numpy()
    e = np.arange(255)[:, None] + np.arange(255)[None, :] - 254 + 4  # 16 ones
    fits = (e >= -100) & (e <= 127)
    assert np.array_equal(got[fits], np.exp2(e[fits].astype(np.float64)))


# ---- grouped products ----
def offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def grouped_ref(qv, qo, bv, bo):
    return [qv[qo[g]:qo[g + 1]] @ bv[bo[g]:bo[g + 1]].T for g in range(len(qo) - 1)]


GROUPS = [
    ([3], [5], 40),
    ([0, 1, 0, 17, 250, 2], [9, 0, 130, 128, 300, 1], 200),
    ([1] * 70, [3] * 70, 64),
    ([0] * 40 + [5, 0, 300], [7] * 40 + [0, 200, 129], 130),
    (list(range(33)), list(range(33, 0, -1)), 96),
    ([2000, 0, 1], [1, 500, 40], 128),
    ([1, 0, 3] * 43, [2, 5, 0] * 43, 32),  # 129 groups
    ([0] * 127 + [1], [1] * 127 + [200], 48),
    ([i % 5 for i in range(700)], [(7 * i) % 23 for i in range(700)], 96),
    ([i % 3 * 150 for i in range(260)], [i % 4 * 100 for i in range(260)], 64),  # several tiles a group
    # many long lists under few queries, some of them without any
    ([i % 5 * 20 for i in range(80)], [1500 + 77 * (i % 40) for i in range(80)], 130),
    ([i % 4 for i in range(120)], [1500 + 177 * (i % 20) for i in range(120)], 96),
]


@pytest.mark.parametrize("mq,mb,dim", GROUPS)
def test_ragged_groups_are_exact(mq, mb, dim):
    qo, bo = offsets(mq), offsets(mb)
    q, qv = exact_codes(int(qo[-1]), dim, 7)
    b, bv = exact_codes(int(bo[-1]), dim, 8)
    bq = BlockQuantizer(dim)
    want = np.concatenate([m.reshape(-1) for m in grouped_ref(qv, qo, bv, bo)])
    tq, tb = torch.from_numpy(qo).cuda(), torch.from_numpy(bo).cuda()
    assert np.array_equal(bq.grouped_product(q, tq, b, tb).double().cpu().numpy(), want)
    assert np.array_equal(bq.grouped_product(q, tq, b, tb, out_size=len(want)).double().cpu().numpy(), want)


@pytest.mark.parametrize("mq,n,dim", [([4], 6, 20), ([0, 3, 250, 0, 1], 200, 300), ([1] * 64, 256, 512),
                                      ([0] * 99 + [7], 33, 64), ([5, 600], 129, 140)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_even_groups(mq, n, dim, kind):
    qo = offsets(mq)
    g = torch.Generator().manual_seed(9)
    bq = BlockQuantizer(dim)
    q = bq.encode(torch.randn((int(qo[-1]), dim), generator=g).to(DTYPES[kind]).cuda())
    b = bq.encode(torch.randn((n * len(mq), dim), generator=g).cuda())
    got = bq.grouped_product(q, torch.from_numpy(qo).cuda(), b, dtype=DTYPES[kind])
    qv, bv = code_values(q), code_values(b)
    bo = np.arange(len(mq) + 1) * n
    ref = np.concatenate(grouped_ref(qv, qo, bv, bo))
    tol = tolerance(ref, np.concatenate(grouped_ref(np.abs(qv), qo, np.abs(bv), bo)), dim, DTYPES[kind])
    assert got.shape == (qo[-1], n) and (np.abs(got.double().cpu().numpy() - ref) <= tol).all()


def test_rows_outside_the_groups_are_left_as_they_were():
    dim, n = 72, 50
    q, qv = exact_codes(30, dim, 10)
    b, bv = exact_codes(3 * n, dim, 11)
    qo = np.array([4, 9, 9, 25], np.int64)
    out = torch.full((30, n), -3.0, device="cuda")
    bq = BlockQuantizer(dim)
    r = [bq._rows(x, True, "x") for x in (q, b)]
    tq = torch.from_numpy(qo).cuda()
    N.call("pxc_bq_grouped_product_device", bq.ctx.handle, C.byref(r[0]), tq.data_ptr(), C.byref(r[1]), None, 3, dim,
           out.data_ptr(), 0, 30 * n, 1)
    bq.check()
    want = np.full((30, n), -3.0)
    for g in range(3):
        want[qo[g]:qo[g + 1]] = qv[qo[g]:qo[g + 1]] @ bv[g * n:(g + 1) * n].T
    assert np.array_equal(out.double().cpu().numpy(), want)
    # ragged, with rows before the first and behind the last group on both sides
    bo = np.array([10, 10, 60, 149], np.int64)
    got = bq.grouped_product(q, tq, b, torch.from_numpy(bo).cuda())
    assert np.array_equal(got.double().cpu().numpy(),
                          np.concatenate([m.reshape(-1) for m in grouped_ref(qv, qo, bv, bo)]))


BAD = [
    ([0, 9, 4, 20], [0, 5, 10, 40], 10**6),  # falls
    ([0, 9, 14, 21], [0, 5, 10, 40], 10**6),  # past the queries
    ([-1, 9, 14, 20], [0, 5, 10, 40], 10**6),  # before the first
    ([0, 9, 14, 20], [0, 5, 10, 41], 10**6),  # past the rows
    ([0, 9, 14, 20], [0, -(2**63), 2**63 - 1, 40], 10**6),
    ([0, 9, 14, 20], [0, 5, 10, 40], 9 * 5 + 5 * 5 + 6 * 30 - 1),  # one value too many
    ([0, 9, 14, 20], [0, 5, 10, 40], 1),
]


@pytest.mark.parametrize("qo,bo,size", BAD)
def test_bad_offsets_are_reported_and_write_nothing_outside(qo, bo, size):
    dim = 48
    q, _ = exact_codes(20, dim, 12)
    b, _ = exact_codes(40, dim, 13)
    bq = BlockQuantizer(dim)
    room = min(size, 9 * 5 + 5 * 5 + 6 * 30)
    out = torch.full((room + 4096,), -9.0, device="cuda")
    r = [bq._rows(x, True, "x") for x in (q, b)]
    tq, tb = torch.tensor(qo, device="cuda"), torch.tensor(bo, device="cuda")
    N.call("pxc_bq_grouped_product_device", bq.ctx.handle, C.byref(r[0]), tq.data_ptr(), C.byref(r[1]), tb.data_ptr(),
           3, dim, out.data_ptr(), 0, room, 1)
    with pytest.raises(Configuration) as e:
        bq.check()
    assert e.value.parameter == "offsets"
    assert (out[room:] == -9).all()
    bq.check()  # reported once
    assert bq.product(q, b).shape == (20, 40)


def test_bad_even_offsets_surface_at_the_next_call():
    dim = 48
    q, _ = exact_codes(20, dim, 12)
    b, _ = exact_codes(40, dim, 13)
    bq = BlockQuantizer(dim)
    bq.grouped_product(q, torch.tensor([0, 30, 20], device="cuda"), b)
    torch.cuda.synchronize()
    with pytest.raises(Configuration):
        bq.product(q, b)
    bq.check()


# ---- the ways of calling ----
def test_host_arrays_give_the_device_results():
    dim = 333
    g = np.random.default_rng(14)
    x, y = g.standard_normal((70, dim)).astype(np.float32), g.standard_normal((210, dim)).astype(np.float16)
    bq = BlockQuantizer(dim)
    hx, hy = bq.encode(x), bq.encode(y)
    dx, dy = bq.encode(torch.from_numpy(x).cuda()), bq.encode(torch.from_numpy(y).cuda())
    assert np.array_equal(hx.codes, dx.codes.cpu().numpy()) and np.array_equal(hy.scales, dy.scales.cpu().numpy())
    assert np.array_equal(bq.decode(hy, dtype=np.float16), bq.decode(dy, dtype=torch.float16).cpu().numpy())
    assert np.array_equal(bq.product(hx, hy), bq.product(dx, dy).cpu().numpy())
    assert np.array_equal(bq.product(hx[3:20], hy[5:100]), bq.product(dx, dy).cpu().numpy()[3:20, 5:100])
    qo, bo = np.array([0, 30, 30, 70]), np.array([0, 10, 100, 210])
    td = [torch.from_numpy(o).cuda() for o in (qo, bo)]
    assert np.array_equal(bq.grouped_product(hx, qo, hy, bo), bq.grouped_product(dx, td[0], dy, td[1]).cpu().numpy())
    assert np.array_equal(bq.grouped_product(hx, qo, hy), bq.grouped_product(dx, td[0], dy).cpu().numpy())
    odd = np.zeros(70 * 336 + 1, np.uint8)[1:].reshape(70, 336)  # host rows at an odd address
    odd[:] = hx.codes
    assert np.array_equal(bq.product(BlockCodes(odd, hx.scales, dim), hy), bq.product(hx, hy))
    with pytest.raises(Configuration):
        bq.grouped_product(hx, np.array([0, 80]), hy, np.array([0, 210]))
    with pytest.raises(Configuration):
        bq.grouped_product(hx, qo, hy, bo, out_size=5)


def test_two_streams_and_two_threads():
    import threading

    dim = 500
    q, qv = exact_codes(150, dim, 15)
    b, bv = exact_codes(2000, dim, 16)
    bq = BlockQuantizer(dim)
    want = qv @ bv.T
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    results[i] = bq.product(q, b)
                torch.cuda.current_stream().synchronize()
        except ProximaError as e:  # pragma: no cover
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for r in results.values():
        assert np.array_equal(r.double().cpu().numpy(), want)


def test_captured_graphs_replay_on_new_values():
    """Two graphs over the same operators, replayed in turn with new inputs and new offsets."""
    dim = 192
    bq = BlockQuantizer(dim)
    x = torch.zeros((60, dim), device="cuda")
    b, bv = exact_codes(400, dim, 17)
    qo, bo = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [None, None]
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        c = bq.encode(x)
        bq.product(c, b)
        bq.grouped_product(c, qo, b, bo, out_size=60 * 400)
    warm.synchronize()
    with torch.cuda.graph(graphs[0]):
        outs[0] = bq.product(bq.encode(x), b)
    with torch.cuda.graph(graphs[1]):
        outs[1] = bq.grouped_product(bq.encode(x), qo, b, bo, out_size=60 * 400)
    for k in range(3):
        g = np.random.default_rng(k)
        v = g.integers(-3, 4, (60, dim)).astype(np.float32)
        v[:, 0] = 3
        o = [np.concatenate([[0], np.sort(g.integers(0, m + 1, 2)), [m]]) for m in (60, 400)]
        x.copy_(torch.from_numpy(v))
        qo.copy_(torch.from_numpy(o[0]))
        bo.copy_(torch.from_numpy(o[1]))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert np.array_equal(outs[0].double().cpu().numpy(), v.astype(np.float64) @ bv.T)
        want = np.concatenate([m.reshape(-1) for m in grouped_ref(v.astype(np.float64), o[0], bv, o[1])])
        assert np.array_equal(outs[1][:len(want)].double().cpu().numpy(), want)
    bq.check()


def test_a_wait_that_runs_out_is_reported_and_leaves_the_device_usable():
    """One group of 224 queries is one tile; its 8,192 blocks take 8,192 * 4 * 112 = 3.7 M cycles at least, more
    than a limit of 1 ms (2 M): the epilogue's wait for it ends, the kernel returns, and the next calls
    say so and work."""
    from proxima_b200.errors import DeviceTimeout
    from proxima_b200.index import Context

    ctx = Context(0)
    dim = 1 << 20
    bq = BlockQuantizer(dim, context=ctx)
    c = BlockCodes(torch.full((224, dim), 0x38, dtype=torch.uint8, device="cuda"),
                   torch.full((224, dim // 128), 127, dtype=torch.uint8, device="cuda"), dim)
    off = torch.tensor([0, 224], device="cuda")
    assert (bq.grouped_product(c, off, c[:128]) == dim).all()
    ctx.set_wait_limit(1)
    bq.grouped_product(c, off, c[:128])
    with pytest.raises(DeviceTimeout):
        bq.check()
    ctx.set_wait_limit(2000)
    assert (bq.grouped_product(c, off, c[:128]) == dim).all()
    assert (bq.product(c, c[:128]) == dim).all()
    bq.check()
    ctx.close()


def test_refusals_on_the_device():
    bq = BlockQuantizer(64)
    c = bq.encode(torch.zeros((8, 64), device="cuda"))
    host = BlockCodes(np.zeros((8, 64), np.uint8), np.zeros((8, 4), np.uint8), 64)
    with pytest.raises(Configuration):
        bq.product(c, host)
    with pytest.raises(Configuration):
        bq.product(host, c)
    with pytest.raises(Configuration):
        bq.encode(torch.zeros((8, 64), device="cuda", dtype=torch.float64))
    with pytest.raises(Configuration):
        bq.product(c, c, out=torch.zeros((8, 9), device="cuda"))
    with pytest.raises(Configuration):
        bq.product(c, c, out=torch.zeros((8, 8), device="cuda").t()[:, ::2])
    with pytest.raises(Configuration):
        bq.grouped_product(c, torch.tensor([0, 8], device="cuda", dtype=torch.int32), c)
    with pytest.raises(Configuration):
        bq.grouped_product(c, [0, 8], c)
    h = bq.ctx.handle
    rows = bq._rows(c, True, "c")
    out = torch.zeros((8, 8), device="cuda")

    def product(q=None, dim=64, ptr=None, dtype=0, stride=8):
        q = q or rows
        N.call("pxc_bq_product_device", h, C.byref(q), C.byref(rows), dim, out.data_ptr() if ptr is None else ptr, dtype, stride, 1)

    R = N.PxcBqRows
    for bad in (dict(dim=0), dict(dim=65), dict(dim=(1 << 20) + 1), dict(dtype=3), dict(dtype=-1), dict(ptr=0),
                dict(ptr=out.data_ptr() + 2), dict(stride=7), dict(stride=1 << 47),
                dict(q=R(rows.codes + 8, rows.scales, 7, 64, 4)), dict(q=R(rows.codes, rows.scales + 1, 7, 64, 4)),
                dict(q=R(rows.codes, rows.scales, 8, 72, 4)), dict(q=R(rows.codes, rows.scales, 8, 48, 4)),
                dict(q=R(rows.codes, rows.scales, 8, 64, 2)), dict(q=R(rows.codes, rows.scales, 8, 64, 0)),
                dict(q=R(None, rows.scales, 8, 64, 4)), dict(q=R(rows.codes, None, 8, 64, 4)),
                dict(q=R(rows.codes, rows.scales, (1 << 31) - 1023, 64, 4))):
        with pytest.raises(Configuration):
            product(**bad)
    product()
    for stride, rws in ((63, rows), (1 << 33, rows)):
        with pytest.raises(Configuration):
            N.call("pxc_bq_encode_device", h, out.data_ptr(), 0, stride, 64, C.byref(rws), 1)
    with pytest.raises(Configuration):
        N.call("pxc_bq_decode_device", h, C.byref(rows), 64, out.data_ptr() + 1, 0, 64, 1)
    off = torch.tensor([0, 8], device="cuda")
    for groups, size, b in ((0, 64, None), (3, 64, None), (1, 63, None), (1, (1 << 48) + 1, off.data_ptr())):
        with pytest.raises(Configuration):
            N.call("pxc_bq_grouped_product_device", h, C.byref(rows), off.data_ptr(), C.byref(rows), b, groups, 64,
                   out.data_ptr(), 0, size, 1)
    with pytest.raises(Configuration):
        N.call("pxc_bq_grouped_product_device", h, C.byref(rows), None, C.byref(rows), None, 1, 64, out.data_ptr(), 0, 64, 1)
    bq.check()


def test_a_run_of_them_together():
    """Vectors encoded once; queries encoded and scored in full and list by list; the best rows are the
    same, and those of the decoded vectors in 64 bits."""
    from proxima_b200 import fixtures

    dim, n, lists = 96, 6000, 40
    data = fixtures.sphere_blobs(n, dim, lists, 21, 22, 0.1)
    queries = fixtures.sphere_blobs(64, dim, lists, 21, 23, 0.1)
    own = np.random.default_rng(24).integers(0, lists, n)
    order = np.argsort(own, kind="stable")
    bo = offsets(np.bincount(own, minlength=lists))
    bq = BlockQuantizer(dim)
    base = bq.encode(torch.from_numpy(data[order]).cuda())
    q = bq.encode(torch.from_numpy(queries).cuda())
    full = bq.product(q, base).cpu().numpy()
    v, w = bq.decode(q).double().cpu().numpy(), bq.decode(base).double().cpu().numpy()
    ref, tol = bound(v, w, torch.float32)
    assert (np.abs(full - ref) <= tol).all()
    best = ref.max(1)
    assert (ref[np.arange(64), full.argmax(1)] >= best - 2 * tol.max()).all()
    # every query probes every list: group g holds all queries, gathered from the same codes
    many = BlockCodes(q.codes.repeat(lists, 1), q.scales.repeat(lists, 1), dim)
    qo = torch.arange(lists + 1, device="cuda") * 64
    flat = bq.grouped_product(many, qo, base, torch.from_numpy(bo).cuda(), out_size=64 * n).cpu().numpy()
    joined = np.concatenate([flat[64 * bo[g]:64 * bo[g + 1]].reshape(64, -1) for g in range(lists)], axis=1)
    assert np.array_equal(joined, full)

"""What the block products do when something goes wrong on the device: who is told, and in what state the
device is left. The failures are offsets that the kernel's checks refuse and waits with a short limit."""
import ctypes as C

import numpy as np
import pytest

from proxima_b200 import _native as N
from proxima_b200.blockquant import BlockCodes, BlockQuantizer
from proxima_b200.errors import Configuration, DeviceTimeout
from proxima_b200.index import Context

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LONG = 1 << 20  # components: 8,192 blocks, so that a tile takes 1 ms at least whatever its width


def ones(rows, dim):
    return BlockCodes(torch.full((rows, dim), 0x38, dtype=torch.uint8, device="cuda"),
                      torch.full((rows, dim // 128), 127, dtype=torch.uint8, device="cuda"), dim)


@pytest.fixture
def ctx():
    c = Context(0)
    yield c
    torch.cuda.synchronize()
    c.close()


# ---- waits that run out ----
@pytest.mark.parametrize("nq,n", [(224, 300), (500, 600), (40, 600)])  # pairs, and single CTAs
def test_a_failed_product_ends_soon_and_leaves_nothing_behind(ctx, nq, n):
    """A tile of 224 queries takes 8,192 * 4 * 112 = 3.7 M cycles at least as a pair of CTAs, one of 176 takes 2.9 M,
    and one of 48 on its own brings 8,192 times 22 KB at 64 bytes a cycle (2.8 M): the epilogue's wait of 1 ms (2 M
    cycles) for it runs out, in either CTA of a pair, while the ring is full of copies. A product of known
    values that starts on the same SMs right behind must not meet them."""
    bq, small = BlockQuantizer(LONG, context=ctx), BlockQuantizer(2048, context=Context.default())
    c = ones(max(nq, n), LONG)
    v = ones(1300, 2048)
    want = bq.product(c[:nq], c[:n])
    assert (want == LONG).all()
    for _ in range(5):
        ctx.set_wait_limit(1)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        bq.product(c[:nq], c[:n])
        end.record()
        after = [small.product(v, v) for _ in range(4)]
        with pytest.raises(DeviceTimeout):
            bq.check()
        # the limit and what was in flight, not a limit for each of the ring's stages
        assert start.elapsed_time(end) < 8.0
        assert all((a == 2048).all() for a in after)
        ctx.set_wait_limit(2000)
        assert torch.equal(bq.product(c[:nq], c[:n]), want)
        bq.check()


# ---- who is told ----
BAD = [0, 30, 20]  # query offsets that fall


def some_codes(bq, rows, seed):
    g = torch.Generator().manual_seed(seed)
    return bq.encode(torch.randint(-3, 4, (rows, bq.dim), generator=g).float().cuda())


def bad_call(bq, q, b):
    bq.grouped_product(q, torch.tensor(BAD, device="cuda"), b)


def test_a_quantiser_hears_of_its_own_calls_alone(ctx):
    a, b = BlockQuantizer(48, context=ctx), BlockQuantizer(48, context=ctx)
    q, base = some_codes(a, 20, 1), some_codes(a, 40, 2)
    want = b.product(q, base)
    bad_call(a, q, base)
    torch.cuda.synchronize()
    # every kind of call of another quantiser on the same context and stream
    x = b.decode(q)
    b.encode(x)
    assert torch.equal(b.product(q, base), want)
    b.grouped_product(q, torch.tensor([0, 5, 20], device="cuda"), base)
    host = b.encode(x.cpu().numpy())
    assert np.array_equal(b.product(host, host), b.product(q, q).cpu().numpy())
    b.check()
    with pytest.raises(Configuration) as e:
        a.check()
    assert e.value.parameter == "offsets"
    a.check()  # once
    # and the one that failed hears of it from each kind of call
    for call in (lambda: a.encode(x), lambda: a.decode(q), lambda: a.product(q, base),
                 lambda: a.grouped_product(q, torch.tensor([0, 20], device="cuda"), base),
                 lambda: a.encode(x.cpu().numpy()), lambda: a.product(host, host)):
        bad_call(a, q, base)
        torch.cuda.synchronize()
        with pytest.raises(Configuration):
            call()
        call()


def test_two_threads_of_which_one_fails(ctx):
    import threading

    rounds = 200
    setup = BlockQuantizer(48, context=ctx)
    q, base = some_codes(setup, 20, 1), some_codes(setup, 40, 2)
    want = setup.product(q, base)
    torch.cuda.synchronize()
    problems, told = [], []

    def bad():
        try:
            bq = BlockQuantizer(48, context=ctx)
            for _ in range(rounds):
                bad_call(bq, q, base)
                try:
                    bq.check()
                except Configuration:
                    told.append(1)
        except BaseException as e:
            problems.append(e)

    def good():
        try:
            bq = BlockQuantizer(48, context=ctx)
            results = []
            for _ in range(rounds):
                results.append(bq.product(q, base))
                bq.check()
            assert len(results) == rounds and all(torch.equal(r, want) for r in results)
        except BaseException as e:
            problems.append(e)

    threads = [threading.Thread(target=f) for f in (bad, good, good)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not problems and len(told) == rounds


def test_calls_on_the_context_are_told_by_stream(ctx):
    bq = BlockQuantizer(48, context=ctx)
    q, base = some_codes(bq, 20, 1), some_codes(bq, 40, 2)
    rq, rb = bq._rows(q, True, "q"), bq._rows(base, True, "b")
    out = torch.zeros(2000, device="cuda")
    off = torch.tensor(BAD, device="cuda")
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()

    def bad(stream):
        N.call("pxc_bq_grouped_product_device", ctx.handle, C.byref(rq), off.data_ptr(), C.byref(rb), None, 2, 48,
               out.data_ptr(), 0, 2000, stream.cuda_stream)

    bad(one)
    torch.cuda.synchronize()
    N.call("pxc_bq_product_device", ctx.handle, C.byref(rq), C.byref(rb), 48, out.data_ptr(), 0, 40, two.cuda_stream)
    N.call("pxc_bq_check", ctx.handle, two.cuda_stream)
    N.call("pxc_bq_check", ctx.handle, None)
    bq.check()
    host = BlockCodes(q.codes.cpu().numpy(), q.scales.cpu().numpy(), 48)
    bq.product(host, host)
    with pytest.raises(Configuration):
        N.call("pxc_bq_check", ctx.handle, one.cuda_stream)
    N.call("pxc_bq_check", ctx.handle, one.cuda_stream)
    bad(one)
    torch.cuda.synchronize()
    with pytest.raises(Configuration):  # the next call there
        N.call("pxc_bq_product_device", ctx.handle, C.byref(rq), C.byref(rb), 48, out.data_ptr(), 0, 40, one.cuda_stream)
    # of a graph, which may run on any stream: any call on the context itself
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=one):
        bad(one)
    with torch.cuda.stream(two):
        graph.replay()
    torch.cuda.synchronize()
    BlockQuantizer(48, context=ctx).product(q, base)
    with pytest.raises(Configuration):
        N.call("pxc_bq_check", ctx.handle, None)


def test_a_host_call_that_fails_says_so_whatever_others_do(ctx):
    """Products of host rows whose wait runs out, beside a thread of calls that succeed on the same context."""
    import threading

    bq = BlockQuantizer(LONG, context=ctx)
    c = BlockCodes(np.full((224, LONG), 0x38, np.uint8), np.full((224, LONG // 128), 127, np.uint8), LONG)
    small = BlockQuantizer(48, context=ctx)
    q = some_codes(small, 20, 1)
    torch.cuda.synchronize()
    stop, problems, calls = threading.Event(), [], []

    def others():
        try:
            while not stop.is_set():
                small.encode(small.decode(q))
                small.check()
                calls.append(1)
        except BaseException as e:
            problems.append(e)

    ctx.set_wait_limit(1)
    t = threading.Thread(target=others)
    t.start()
    try:
        for _ in range(8):
            with pytest.raises(DeviceTimeout):
                bq.product(c, c)
    finally:
        stop.set()
        t.join()
        ctx.set_wait_limit(2000)
    assert not problems and calls
    bq.check()
    assert (bq.product(c[:3], c) == LONG).all()


def test_two_kinds_of_failure_are_both_told(ctx):
    bq = BlockQuantizer(LONG, context=ctx)
    c = ones(224, LONG)
    small = BlockCodes(c.codes[:40], c.scales[:40], LONG)
    bq.product(small, small)
    graph = torch.cuda.CUDAGraph()  # as no call may come between the two
    off, whole = torch.tensor([0, 30, 20], device="cuda"), torch.tensor([0, 224], device="cuda")
    ctx.set_wait_limit(1)
    with torch.cuda.graph(graph):
        bq.grouped_product(small, off, small)
        bq.grouped_product(c, whole, c)
    ctx.set_wait_limit(2000)
    graph.replay()
    with pytest.raises(DeviceTimeout):
        bq.check()
    with pytest.raises(Configuration):
        bq.check()
    bq.check()


def test_graphs_report_to_the_quantiser_that_was_captured(ctx):
    a, b = BlockQuantizer(48, context=ctx), BlockQuantizer(48, context=ctx)
    q, base = some_codes(a, 20, 1), some_codes(a, 40, 2)
    off = torch.tensor([0, 10, 20], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.grouped_product(q, off, base)
    graph.replay()
    a.check()
    off.copy_(torch.tensor(BAD))
    with torch.cuda.stream(torch.cuda.Stream()):
        graph.replay()
        torch.cuda.synchronize()
    b.check()
    with pytest.raises(Configuration):
        a.product(q, base)


def test_failures_of_quantisers_that_are_gone(ctx):
    """Their work may still run. No other quantiser's calls are told of it, but whoever checks is."""
    kept = BlockQuantizer(48, context=ctx)
    q, base = some_codes(kept, 20, 1), some_codes(kept, 40, 2)
    want = kept.product(q, base)
    for i in range(3000):
        bad_call(BlockQuantizer(48, context=ctx), q, base)
        if i % 100 == 0:
            later = BlockQuantizer(48, context=ctx)
            assert torch.equal(later.product(q, base), want) and torch.equal(kept.product(q, base), want)
    told = 0
    for _ in range(3001):
        try:
            BlockQuantizer(48, context=ctx).check()
            break
        except Configuration:
            told += 1
    assert 1 <= told <= 3000
    kept.check()
    # a graph that outlives the quantiser it was captured with
    off = torch.tensor([0, 10, 20], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        BlockQuantizer(48, context=ctx).grouped_product(q, off, base)
    for _ in range(1500):  # more than there are records before they are given out again
        BlockQuantizer(48, context=ctx).product(q, base)
    off.copy_(torch.tensor(BAD))
    kept.check()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept.product(q, base), want)
    with pytest.raises(Configuration):
        kept.check()
    kept.check()


def test_a_closed_context_is_refused():
    ctx = Context(0)
    bq = BlockQuantizer(48, context=ctx)
    q = some_codes(bq, 20, 1)
    torch.cuda.synchronize()
    ctx.close()
    for call in (lambda: bq.decode(q), lambda: bq.product(q, q), bq.check,
                 lambda: BlockQuantizer(48, context=ctx).decode(q)):
        with pytest.raises(Configuration):
            call()


# ---- offsets ----
def test_groups_behind_a_bad_one_do_no_work(ctx):
    """Offsets that go up and down: every other group would pair all queries with its rows. Only those before the
    first fall count, so the work is that of one group and not that of half a million (45 million tiles)."""
    groups, nq, dim = 1 << 20, 20_000, 16
    bq = BlockQuantizer(dim, context=ctx)
    q, base = some_codes(bq, nq, 1), some_codes(bq, groups, 2)
    off = torch.zeros(groups + 1, dtype=torch.int64, device="cuda")
    bq.grouped_product(q, off, base)
    off[1::2] = nq
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = bq.grouped_product(q, off, base)
    end.record()
    with pytest.raises(Configuration):
        bq.check()
    assert start.elapsed_time(end) < 30.0
    assert got.shape == (nq, 1)


@pytest.mark.parametrize("bad", [0, 1, 3, 4, 127, 128, 131, 300, 511])
@pytest.mark.parametrize("ragged", [False, True])
def test_groups_before_a_bad_one_are_whole_and_those_behind_are_not_written(ctx, bad, ragged):
    """512 groups of 3 queries and 2 rows, of which one has offsets that fall."""
    groups, dim = 512, 32
    bq = BlockQuantizer(dim, context=ctx)
    q, base = some_codes(bq, 3 * groups, 3), some_codes(bq, 2 * groups, 4)
    r = [bq._rows(x, True, "x") for x in (q, base)]
    qo, bo = 3 * torch.arange(groups + 1), 2 * torch.arange(groups + 1)
    good = bq.grouped_product(q, qo.cuda(), base).reshape(-1)
    qo[bad + 1:] += 5
    qo[bad] += 9  # past its end
    out = torch.full((6 * groups,), -9.0, device="cuda")
    dqo, dbo = qo.cuda(), bo.cuda()
    N.call("pxc_bq_grouped_product_device", ctx.handle, C.byref(r[0]), dqo.data_ptr(), C.byref(r[1]),
           dbo.data_ptr() if ragged else None, groups, dim, out.data_ptr(), 0, 6 * groups, 1)
    with pytest.raises(Configuration):
        bq.check()
    before = max(bad - 1, 0)  # the group before ends 9 queries later
    assert torch.equal(out[:6 * before], good[:6 * before])
    written = 6 * before + (2 * 12 if bad else 0)
    assert (out[written:] == -9).all()


@pytest.mark.parametrize("nq,n,qo,bo,size", [
    (0, 6, [0, 2], None, 0),  # no queries: past them
    (0, 6, [0, 0, 0], [0, 7, 6], 0),
    (5, 0, [0, 6], None, 0),  # no rows
    (5, 0, [3, 2, 5], [0, 0, 0], 0),
    (5, 0, [0, 5], [0, 1], 9),
    (5, 6, [0, 5], [0, 6], 0),  # no room
    (5, 6, [0, 0, 5], [0, 4, 6], 0),
    (5, 6, [0] * 700 + [5], [0] * 700 + [6], 0),
])
def test_bad_offsets_of_an_empty_product_are_told_too(ctx, nq, n, qo, bo, size):
    bq = BlockQuantizer(48, context=ctx)
    q, b = bq.encode(torch.ones((nq, 48), device="cuda")), bq.encode(torch.ones((n, 48), device="cuda"))
    r = [bq._rows(x, True, "x") for x in (q, b)]
    off = [o and torch.tensor(o, device="cuda") for o in (qo, bo)]
    out = torch.full((64,), -9.0, device="cuda")
    N.call("pxc_bq_grouped_product_device", ctx.handle, C.byref(r[0]), off[0].data_ptr(), C.byref(r[1]), N.ptr(off[1]),
           len(qo) - 1, 48, out.data_ptr(), 0, size, 1)
    with pytest.raises(Configuration) as e:
        bq.check()
    assert e.value.parameter == "offsets" and (out == -9).all()
    if bo is not None:
        bq.grouped_product(q, off[0], b, off[1], out_size=size)
        with pytest.raises(Configuration):
            bq.check()


@pytest.mark.parametrize("nq,n,qo,bo,size", [
    (0, 6, [0, 0, 0], None, 0), (0, 6, [0, 0], [2, 5], 0), (5, 0, [1, 4], None, 0), (5, 0, [0, 5], [0, 0], 7),
    (5, 6, [0, 0, 5], [0, 4, 4], 0),
])
def test_good_offsets_of_an_empty_product_are_no_failure(ctx, nq, n, qo, bo, size):
    bq = BlockQuantizer(48, context=ctx)
    q, b = bq.encode(torch.ones((nq, 48), device="cuda")), bq.encode(torch.ones((n, 48), device="cuda"))
    off = [o and torch.tensor(o, device="cuda") for o in (qo, bo)]
    bq.grouped_product(q, off[0], b, off[1], out_size=None if bo is None else size)
    bq.check()

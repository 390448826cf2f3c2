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

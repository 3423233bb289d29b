"""Products whose tiles are narrow and more than the SMs, so that a CTA takes several with both of its accumulators."""
import pytest
import torch

import flow_b200 as fb
from test_gpu_product import HALF, check, operands, ragged, wants

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k,groups", [(4, 32768, 1024, 1), (16, 50000, 512, 1), (1, 30000, 64, 1), (5, 40008, 256, 1), (13, 20008, 520, 1),
                                          (4, 1024, 32768, 1), (16, 512, 50000, 1), (7, 264, 40008, 1), (2, 128, 30000, 1),
                                          (40, 1024, 256, 40), (300, 2048, 128, 64)])
def test_few_rows_and_many_channels(ctx, m, n, k, groups, dtype):
    """Whole numbers, bit for bit: 16 columns and 235 to 391 tiles of 128 lanes, forward (n large) and for the rows'
    gradient (k large), with rows on 16-byte boundaries and, the outputs alone, off them."""
    check(ctx, m, n, k, groups, dtype)
    check(ctx, m, n, k, groups, dtype, opads=(3, 5, 0), seed=5)


@pytest.mark.parametrize("m,n,k,groups,pads", [(1500, 516, 771, 11, (0, 0, 0)), (1500, 520, 776, 11, (8, 0, 8)), (1500, 520, 771, 11, (0, 0, 0)),
                                               (1501, 517, 776, 11, (0, 0, 0)), (900, 1029, 2051, 1, (0, 0, 0)), (2000, 768, 768, 60, (0, 0, 0))])
def test_copied_operands_and_last_blocks_many_times(ctx, m, n, k, groups, pads):
    """What one CTA of a pair writes to its shared memory is read by the other's products: copied blocks, and last blocks
    whose rows of the next group are cleared. Forty passes, each from other contents of shared memory, bit for bit."""
    dtype = torch.bfloat16
    sets = [operands(m, n, k, groups, dtype, pads=pads, seed=s) for s in (1, 11)]
    off = ragged(m, groups, 3) if groups > 1 else None
    site = fb.product_site(m, n, k, dtype, groups=groups, ldx=sets[0][0].ld, ldw=sets[0][1].ld, lddy=sets[0][2].ld)
    want = []
    for x, w, dy in sets:
        y, dx, dw = wants(x.t, w.t.reshape(groups, n, k), dy.t, off)
        want.append((y.to(dtype), dx.to(dtype), dw.to(dtype)))
    y, dx, dw = (torch.empty(s, dtype=dtype, device="cuda") for s in ((m, n), (m, k), (groups, n, k)))
    for i in range(40):
        x, w, dy = sets[i % 2]
        ctx.product(site, x.t, w.t, y, offsets=off)
        ctx.product_grad(site, x.t, w.t, dy.t, dx, dw, offsets=off)
        for got, right, what in zip((y, dx, dw), want[i % 2], ("y", "dx", "dw")):
            assert torch.equal(got, right), (i, what)

"""Products whose tiles are narrow and more than the SMs, so that a CTA takes several with both of its accumulators."""
import pytest
import torch

import flow_b200 as fb
from test_gpu_product import HALF, check

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

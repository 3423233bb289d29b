"""Calls that come down to zeros or to a copy, at strides that only they could not take: dropout of everything, and the
gradient of the loss of no rows."""
import pytest
import torch

import flow_b200 as fb
from _rows import TYPES, Guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [True, False])
def test_one_row_has_any_stride(ctx, residual, dtype):
    """A single row's stride is not used, here one below its length."""
    x, rng = torch.full((1, 100), float("nan"), dtype=dtype, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    r = torch.arange(100, device="cuda").to(dtype)[None] if residual else None
    y = Guarded(1, 100, dtype)
    for p in (1.0, 0.0):
        ctx.dropout(fb.dropout_site(1, 100, dtype, p, ldx=1, ldr=1, ldy=1), x, r, y.t, rng)
        assert torch.equal(y.t, r if residual else torch.zeros_like(y.t)) if p else torch.isnan(y.t).all()
    assert y.intact()
    w = Guarded(1, 40, torch.bfloat16)
    w.t.fill_(3)
    e = torch.zeros(0, device="cuda")
    ctx.linear_loss_grad(fb.loss_site(0, 1, 40, torch.bfloat16, lddw=1), e.bfloat16().view(0, 40), None, e.int(), e, e, None, w.t, None)
    assert not w.t.any() and w.intact()


@pytest.mark.parametrize("rows", [1, 3])
def test_rows_in_a_row_and_apart(ctx, rows):
    for pads in ((0, 0), (3, 0), (0, 5), (8, 8)):
        r, y = Guarded(rows, 70, torch.float16, pads[0]).put(torch.randn(rows, 70, device="cuda")), Guarded(rows, 70, torch.float16, pads[1])
        rng = torch.zeros(2, dtype=torch.int64, device="cuda")
        for res in (r, None):
            y.t.fill_(5)
            site = fb.dropout_site(rows, 70, torch.float16, 1.0, ldx=r.ld, ldr=r.ld, ldy=y.ld)
            ctx.dropout(site, r.t, res.t if res else None, y.t, rng)
            assert torch.equal(y.t, r.t if res else torch.zeros_like(r.t)) and y.intact()


def test_strides_of_more_than_two_gigabytes(ctx):
    ld = (1 << 29) + 8
    a, b = (torch.full((2 * ld + 24,), v, device="cuda") for v in (2.0, 7.0))
    r, y = (t[:2 * ld + 24].as_strided((3, 24), (ld, 1)) for t in (a, b))
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    r.copy_(torch.randn(3, 24, device="cuda"))
    for res in (r, None):
        for p in (1.0, 0.5):
            ctx.dropout(fb.dropout_site(3, 24, torch.float32, p, ldx=ld, ldr=ld, ldy=ld), r, res, y, rng)
            if p == 1.0:
                assert torch.equal(y, r if res is not None else torch.zeros_like(r))
    assert b[24] == 7 and b[ld - 1] == 7 and b[ld + 24] == 7 and b[2 * ld - 1] == 7
    half = b.view(torch.bfloat16)  # rows at 2 * ld of its elements
    w = half.as_strided((3, 8), (2 * ld, 1))
    w.fill_(3)
    e = torch.zeros(0, device="cuda")
    ctx.linear_loss_grad(fb.loss_site(0, 3, 8, torch.bfloat16, lddw=2 * ld), e.bfloat16().view(0, 8), None, e.int(), e, e, None, w, None)
    assert not w.any() and half[2 * ld - 1] != 0

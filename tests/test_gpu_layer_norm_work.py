"""The gradient of layer norm writes nothing behind the scratch that it asks for, on a B200: `work` is the first
bytes of a longer buffer whose rest holds a marker."""
import pytest
import torch

import flow_b200 as fb
from _rows import TYPES, assert_within
from test_gpu_layer_norm import grad_formula, rows_of

pytestmark = pytest.mark.gpu
EPS, MARK, TAIL = 1e-5, 0xA5, 4096


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def grad(ctx, x, dy, dx, wide=0):
    """dw and db (rows at stride d + wide), and the marker looked at."""
    rows, d = x.shape
    ld = d + wide
    site = fb.norm_site(rows, d, x.dtype, wdtype=torch.float32, eps=EPS, ldx=ld, ldy=ld, lddy=ld, lddx=ld)
    n = ctx.layer_norm_grad_workspace(site)
    buf = torch.full((n + TAIL,), MARK, dtype=torch.uint8, device="cuda")
    mean, rstd = x.float().mean(1), torch.full((rows,), 0.7, device="cuda")  # any values: the gradient takes them as given
    dw, db = (torch.full((d,), float("nan"), device="cuda") for _ in range(2))
    w = rows_of(1, d, torch.float32, 9)[0]
    ctx.layer_norm_grad(site, x, w, mean, rstd, dy, dx, dw, db, buf[:n])
    assert (buf[n:] == MARK).all(), "written behind work"
    return w, mean, rstd, dw, db


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 2, 7, 9, 57, 73, 125, 253, 1021, 1024, 2039, 2050, 8187, 8193, 20001])
def test_sums_over_no_rows(ctx, d, dtype):
    """Widths that no pack divides: with V columns a pack, whole packs would end up to V - 1 floats behind the last row
    of partial sums."""
    x = torch.empty(0, d, dtype=dtype, device="cuda")
    _, _, _, dw, db = grad(ctx, x, x, x)
    assert not dw.any() and not db.any() and not torch.isnan(dw).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d,wide", [
    (1, 9, 0), (1, 1021, 0), (9, 121, 7),                                      # a block for each class of rows
    (1300, 57, 0), (20011, 61, 3), (1500, 128, 0), (3000, 127, 1),             # groups of lanes
    (600, 505, 0), (400, 1024, 0), (700, 2039, 2), (300, 4096, 0), (160, 8185, 0), (150, 8192, 0),
    (1, 8200, 0), (40, 9001, 0), (70, 16384, 0), (3, 40003, 1), (200, 33000, 0),  # longer rows: sums by column
])
def test_every_kind_of_sums(ctx, rows, d, wide, dtype):
    a, b, c = (torch.zeros(rows, d + wide, device="cuda").to(dtype)[:, :d] for _ in range(3))
    a.copy_(rows_of(rows, d, dtype, 1))
    b.copy_(rows_of(rows, d, dtype, 2))
    w, mean, rstd, dw, db = grad(ctx, a, b, c, wide)
    _, gw, gb, _, gw_err, gb_err = grad_formula(a, w, mean, rstd, b)
    assert_within(dw, gw, gw_err, "dw")
    assert_within(db, gb, gb_err, "db")

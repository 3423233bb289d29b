"""Products and the loss where an output is one of the operands: refused on the host (without a GPU, as in
test_training_refusals.py) wherever the call reads it, right where it does not."""
import pytest
import torch

import flow_b200 as fb
from test_gpu_linear_loss import inputs
from test_gpu_product import wants, whole
from test_rows_refusals import ACCEPTED, INVALID, P
from test_training_refusals import loss_grad, product, product_grad, small


def test_products_refuse_outputs_that_are_operands():
    s = small()
    for kw in (dict(y=P), dict(y=2 * P)):
        assert product(s, **kw) == (INVALID, "y is x or w")
    for kw in (dict(dx=P), dict(dx=2 * P), dict(dx=4 * P), dict(dw=P), dict(dw=2 * P), dict(dw=4 * P), dict(dx=4 * P, dw=None),
               dict(dw=4 * P, dx=None), dict(dw=P, dx=None), dict(dx=2 * P, dw=None)):
        rc, msg = product_grad(s, **kw)
        assert rc == INVALID and "reads" in msg, (kw, msg)
    assert product_grad(s, dx=P, dw=None) == ACCEPTED and product_grad(s, dw=2 * P, dx=None) == ACCEPTED


def test_the_loss_refuses_outputs_that_are_operands():
    s = fb.loss_site(7, 5, 3, "bfloat16")
    for kw in (dict(dh=2 * P), dict(dw=P), dict(dw=2 * P), dict(dw=7 * P), dict(dw=P, dh=None), dict(dh=2 * P, dw=None)):
        rc, msg = loss_grad(s, **kw)
        assert rc == INVALID and "reads" in msg, (kw, msg)
    assert loss_grad(fb.loss_site(7, 5, 3, "bfloat16", lddh=4), dh=P)[0] == INVALID
    assert loss_grad(s, dh=P) == ACCEPTED and loss_grad(s, dw=2 * P, dh=None) == ACCEPTED


@pytest.mark.gpu
def test_outputs_in_place_of_what_is_not_read():
    ctx, t = fb.Context((0,)), torch.bfloat16
    m, n, k = 300, 72, 136
    x, w, dy = whole((m, k), t, 1), whole((1, n, k), t, 2), whole((m, n), t, 3)
    _, wdx, wdw = wants(x, w, dy, None)
    site = fb.product_site(m, n, k, t)
    dx, dw = x.clone(), w.clone()
    ctx.product_grad(site, dx, w, dy, dx, None)
    ctx.product_grad(site, x, dw, dy, None, dw)
    assert torch.equal(dx, wdx.to(t)) and torch.equal(dw, wdw.to(t))
    h, w, targets, dloss = inputs(300, 700, 72, t, 3, 0.2)
    site = fb.loss_site(300, 700, 72, t)
    work = torch.empty(ctx.linear_loss_workspace(site), dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(300, device="cuda") for _ in range(2))
    ctx.linear_loss(site, h.t, w.t, targets, loss, lse, work)
    dh, dw = torch.empty(300, 72, dtype=t, device="cuda"), torch.empty(700, 72, dtype=t, device="cuda")
    ctx.linear_loss_grad(site, h.t, w.t, targets, lse, dloss, dh, dw, work)
    h2, w2 = h.t.clone(), w.t.clone()
    dw2 = torch.empty_like(dw)
    ctx.linear_loss_grad(site, h2, w.t, targets, lse, dloss, h2, dw2, work)
    assert torch.equal(h2, dh) and torch.equal(dw2, dw)
    ctx.linear_loss_grad(site, h.t, w2, targets, lse, dloss, None, w2, work)
    assert torch.equal(w2, dw)
    ctx.close()

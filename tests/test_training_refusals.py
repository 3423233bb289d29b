"""What the products, the loss and dropout refuse, without a GPU: as in test_rows_refusals.py, every record and pointer
is checked before the context is looked at, so a call with no context tells a refusal from an accepted call, and the
Python wrappers' checks are tested with CPU tensors on a context object that drives no device."""
import ctypes

import pytest
import torch

import flow_b200 as fb
from test_rows_refusals import ACCEPTED, INVALID, P, UNSUPPORTED, call, with_

F, H, I, L = torch.float32, torch.bfloat16, torch.int32, torch.int64


@pytest.fixture
def ctx():
    c = fb.Context.__new__(fb.Context)
    c._h, c.devices = None, [-1]
    return c


def product(site, x=P, w=2 * P, off=3 * P, y=4 * P):
    return call("product", site, x, w, off, y)


def product_grad(site, x=P, w=2 * P, off=3 * P, dy=4 * P, dx=5 * P, dw=6 * P):
    return call("product_grad", site, x, w, off, dy, dx, dw)


def loss(site, h=P, w=2 * P, t=3 * P, out=4 * P, lse=5 * P, work=6 * P, n=1 << 40):
    return call("linear_loss", site, h, w, t, out, lse, work, n)


def loss_grad(site, h=P, w=2 * P, t=3 * P, lse=5 * P, g=None, dh=7 * P, dw=8 * P, work=6 * P, n=1 << 40):
    return call("linear_loss_grad", site, h, w, t, lse, g, dh, dw, work, n)


def dropout(site, x=P, r=2 * P, rng=3 * P, y=4 * P):
    return call("dropout", site, x, r, rng, y)


def small(**kw):
    return with_(fb.product_site(7, 5, 3, "bfloat16", groups=2), **kw)


def test_accepted():
    for t in ("float16", "bfloat16"):
        for wide in (None, "float32"):
            s = fb.product_site(7, 5, 3, t, groups=2, ytype=wide, dwtype=wide)
            assert product(s) == ACCEPTED and product_grad(s) == ACCEPTED
        assert product(fb.product_site(7, 5, 3, t), off=None) == ACCEPTED
        assert product_grad(fb.product_site(7, 5, 3, t), off=None, dx=None, w=None) == ACCEPTED
        assert product_grad(fb.product_site(7, 5, 3, t), off=None, dw=None, x=None) == ACCEPTED
        s = fb.loss_site(7, 5, 3, t)
        assert loss(s) == ACCEPTED and loss(s, lse=None) == ACCEPTED and loss_grad(s) == ACCEPTED
        assert loss_grad(s, dh=None) == ACCEPTED and loss_grad(s, dw=None) == ACCEPTED
    for t in ("float32", "float16", "bfloat16"):
        for p in (0.0, 0.5, 1.0):
            assert dropout(fb.dropout_site(7, 5, t, p)) == ACCEPTED
    assert dropout(fb.dropout_site(7, 5, "float32", 0.1), r=None) == ACCEPTED


def test_nothing_to_do():
    assert product(fb.product_site(0, 5, 3, "float16"), x=None, y=None, off=None)[0] == 0
    assert product(fb.product_site(7, 0, 3, "float16"), w=None, y=None, off=None)[0] == 0
    assert product_grad(fb.product_site(7, 5, 3, "float16"), dx=None, dw=None, off=None)[0] == 0
    assert loss(fb.loss_site(0, 5, 3, "float16"), h=None, t=None, out=None)[0] == 0
    assert loss_grad(fb.loss_site(7, 5, 3, "float16"), dh=None, dw=None)[0] == 0
    assert dropout(fb.dropout_site(0, 5, "float16", 0.1), x=None, y=None)[0] == 0


@pytest.mark.parametrize("f", [product, product_grad])
@pytest.mark.parametrize("change,rc,text", [
    (dict(dtype=0), INVALID, "f16 or bf16"), (dict(dtype=3), INVALID, "f16 or bf16"), (dict(dtype=-1), INVALID, "f16 or bf16"),
    (dict(ytype=1), INVALID, "rows' type"), (dict(dwtype=3), INVALID, "rows' type"),
    (dict(groups=0), INVALID, "groups"), (dict(groups=65536), INVALID, "groups"),
    (dict(m=1 << 31), UNSUPPORTED, "2^31"), (dict(n=1 << 31), UNSUPPORTED, "2^31"), (dict(k=1 << 31), UNSUPPORTED, "2^31"),
])
def test_products_refuse_the_record(f, change, rc, text):
    got, msg = f(small(**change))
    assert got == rc and text in msg, msg


@pytest.mark.parametrize("f,change", [(product, "ldx"), (product, "ldw"), (product, "ldy"), (product_grad, "ldx"),
                                      (product_grad, "ldw"), (product_grad, "lddy"), (product_grad, "lddx"), (product_grad, "lddw")])
@pytest.mark.parametrize("ld", [2, 1 << 61])
def test_products_refuse_strides(f, change, ld):
    rc, msg = f(small(**{change: ld}))
    assert rc == INVALID and "stride" in msg, msg


@pytest.mark.parametrize("f,change", [(product, "ldg"), (product_grad, "ldg"), (product_grad, "lddg")])
def test_products_refuse_overlapping_matrices(f, change):
    rc, msg = f(small(**{change: 14}))
    assert rc == INVALID and "between groups" in msg, msg


def test_products_refuse_pointers():
    s = small()
    for kw in (dict(x=None), dict(w=None), dict(y=None)):
        assert product(s, **kw)[1] == "null x, w or y"
    for kw in (dict(x=P + 1), dict(w=P + 1), dict(y=P + 1), dict(off=P + 2)):
        assert "aligned" in product(s, **kw)[1]
    assert product(s, off=None)[1] == "several groups need offsets" == product_grad(s, off=None)[1]
    for kw in (dict(x=None), dict(w=None), dict(dy=None)):
        assert product_grad(s, **kw)[1] == "null x, w or dy"
    for kw in (dict(x=P + 1), dict(w=P + 1), dict(dy=P + 1), dict(dx=P + 1), dict(dw=P + 1), dict(off=P + 2)):
        assert "aligned" in product_grad(s, **kw)[1]
    assert "aligned" in product(with_(small(), ytype=0), y=P + 2)[1]
    assert product(None)[0] == product_grad(None)[0] == INVALID


@pytest.mark.parametrize("f", [loss, loss_grad])
@pytest.mark.parametrize("change,rc,text", [
    (dict(dtype=0), INVALID, "f16 or bf16"), (dict(vocab=0), INVALID, "vocabulary"), (dict(d=0), INVALID, "vocabulary"),
    (dict(rows=1 << 31), UNSUPPORTED, "2^31"), (dict(vocab=1 << 31), UNSUPPORTED, "2^31"), (dict(d=1 << 31), UNSUPPORTED, "2^31"),
    (dict(ldh=2), INVALID, "stride"), (dict(ldw=2), INVALID, "stride"), (dict(lddh=2), INVALID, "stride"),
    (dict(lddw=2), INVALID, "stride"), (dict(ldw=1 << 37), UNSUPPORTED, "2^38"),
])
def test_losses_refuse_the_record(f, change, rc, text):
    got, msg = f(with_(fb.loss_site(7, 5, 3, "bfloat16"), **change))
    assert got == rc and text in msg, msg


def test_losses_refuse_pointers():
    s = fb.loss_site(7, 5, 3, "bfloat16")
    for kw in (dict(h=None), dict(w=None), dict(t=None), dict(out=None)):
        assert "null" in loss(s, **kw)[1]
    for kw in (dict(h=P + 1), dict(w=P + 1), dict(t=P + 2), dict(out=P + 2), dict(lse=P + 2)):
        assert "aligned" in loss(s, **kw)[1]
    for kw in (dict(h=None), dict(w=None), dict(t=None), dict(lse=None)):
        assert "null" in loss_grad(s, **kw)[1]
    for kw in (dict(dh=P + 1), dict(dw=P + 1), dict(g=P + 2), dict(t=P + 2)):
        assert "aligned" in loss_grad(s, **kw)[1]
    n = ctypes.c_uint64()
    assert call("linear_loss_workspace", s, None, 1, None) == (INVALID, "bytes is null")
    assert call("linear_loss_workspace", s, None, 1, ctypes.byref(n)) == ACCEPTED
    assert loss(None)[0] == loss_grad(None)[0] == INVALID


@pytest.mark.parametrize("change,rc,text", [
    (dict(dtype=3), INVALID, "f32, f16 or bf16"), (dict(p=-0.1), INVALID, "p is"), (dict(p=1.01), INVALID, "p is"),
    (dict(p=float("nan")), INVALID, "p is"), (dict(rows=1 << 31), UNSUPPORTED, "2^31"), (dict(d=1 << 31), UNSUPPORTED, "2^31"),
    (dict(ldx=4), INVALID, "stride"), (dict(ldr=4), INVALID, "stride"), (dict(ldy=4), INVALID, "stride"),
])
def test_dropout_refuses_the_record(change, rc, text):
    got, msg = dropout(with_(fb.dropout_site(7, 5, "bfloat16", 0.5), **change))
    assert got == rc and text in msg, msg


def test_dropout_refuses_pointers():
    s = fb.dropout_site(7, 5, "bfloat16", 0.5)
    for kw in (dict(x=None), dict(y=None), dict(rng=None)):
        assert "null" in dropout(s, **kw)[1]
    for kw in (dict(x=P + 1), dict(r=P + 1), dict(y=P + 1), dict(rng=P + 4)):
        assert "aligned" in dropout(s, **kw)[1]
    s = fb.dropout_site(7, 5, "bfloat16", 0.5, ldy=6)
    assert "same stride" in dropout(s, y=P)[1] and "same stride" in dropout(s, y=2 * P)[1]
    assert dropout(None)[0] == INVALID


def cases():
    z, h = torch.zeros, lambda *s: torch.zeros(*s, dtype=H)
    off, t, rng = z(3, dtype=I), z(7, dtype=I), z(2, dtype=L)
    p, s = fb.product_site(7, 5, 3, H, groups=2), fb.loss_site(7, 5, 3, H)
    return {
        "product": (p, [h(7, 3), h(2, 5, 3), h(7, 5), off]),
        "product_grad": (p, [h(7, 3), h(2, 5, 3), h(7, 5), h(7, 3), h(2, 5, 3), off]),
        "linear_loss": (s, [h(7, 3), h(5, 3), t, z(7), z(7), z(64)]),
        "linear_loss_grad": (s, [h(7, 3), h(5, 3), t, z(7), z(7), h(7, 3), h(5, 3), z(64)]),
        "dropout": (fb.dropout_site(7, 5, H, 0.5), [h(7, 5), h(7, 5), h(7, 5), rng]),
    }


@pytest.mark.parametrize("name", cases())
def test_methods_and_direct_calls(ctx, name):
    """Plain tensors reach the C entry, through the binding and through ctypes; a wrong type, a shorter tensor and
    another device do not."""
    assert set(cases()) == set(fb._Direct.TRAINING)
    site, args = cases()[name]
    with pytest.raises(fb.MapalInfraError, match="ctx is null|aligned"):
        getattr(ctx, name)(site, *args)  # binds the direct calls
    direct, h = getattr(fb._direct, name), ctypes.c_void_p()
    assert direct(h, -1, site, *args) == INVALID
    assert direct(h, 0, site, *args) is None and direct(h, -1, None, *args) is None
    assert direct(h, -1, site, *args[:-1]) is None and direct() is None
    for k, t in enumerate(args):
        work = name.startswith("linear") and k == len(args) - 1
        bad = [t.double()] if not work else []
        bad += [t.flatten()[:-1]] if not work else []
        for b in bad:
            assert direct(h, -1, site, *args[:k], b, *args[k + 1:]) is None, (name, k)
            with pytest.raises(ValueError):
                getattr(ctx, name)(site, *args[:k], b, *args[k + 1:])
        wide = torch.stack([t, t], -1)[..., 0]  # every second element
        with pytest.raises(ValueError):
            getattr(ctx, name)(site, *args[:k], wide, *args[k + 1:])
    ctx.devices = [0]
    with pytest.raises(ValueError, match="the context drives"):
        getattr(ctx, name)(site, *args)


@pytest.mark.parametrize("name", cases())
def test_slices_are_as_long_as_they_are(ctx, name):
    site, args = cases()[name]
    for k, t in enumerate(args):
        if t.dim() == 2:
            long = torch.zeros(2 * t.size(0), t.size(1), dtype=t.dtype)[:t.size(0) - 1]
            with pytest.raises(ValueError, match="holds"):
                getattr(ctx, name)(site, *args[:k], long, *args[k + 1:])


def test_matrices_of_products(ctx):
    site = fb.product_site(7, 5, 3, H, groups=2, ldw=4, ldg=24)
    x, y, off = torch.zeros(7, 3, dtype=H), torch.zeros(7, 5, dtype=H), torch.zeros(3, dtype=I)
    w = torch.zeros(3, 6, 4, dtype=H)
    with pytest.raises(fb.MapalInfraError, match="ctx is null|aligned"):
        ctx.product(site, x, w[:2, :5, :3], y, offsets=off)
    for bad in (w[:1, :5, :3], w[:2, :4, :3], w[:2, :5, :2]):
        with pytest.raises(ValueError, match="^w "):
            ctx.product(site, x, bad, y, offsets=off)


def test_scratch_of_the_loss(ctx):
    site, args = cases()["linear_loss"]
    for bad in (torch.empty(1, dtype=torch.uint8).expand(1 << 20), torch.empty(64)[::2]):
        with pytest.raises(ValueError, match="work must be contiguous"):
            ctx.linear_loss(site, *args[:-1], bad)


def test_record_sizes():
    """As the header has them: eleven 64-bit and four 32-bit fields, and so on."""
    assert ctypes.sizeof(fb.ProductSite) == 11 * 8 + 4 * 4
    assert ctypes.sizeof(fb.LossSite) == 7 * 8 + 2 * 4
    assert ctypes.sizeof(fb.DropoutSite) == 6 * 8 + 2 * 4

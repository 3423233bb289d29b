"""What the row-wise operators refuse, without a GPU: every record and pointer
is checked before the context is looked at, so a call with no context tells a
refusal (its message) from an accepted call ("ctx is null"). The Python
wrappers' checks of tensors are tested with CPU tensors on a context object
that drives no device."""
import ctypes

import pytest
import torch

import flow_b200 as fb

INVALID, UNSUPPORTED = fb.ERR_INVALID, fb.ERR_UNSUPPORTED
P = 1 << 20  # an address that no call gets as far as reading


def call(name, site, *args):
    L = fb.lib()
    rc = getattr(L, "mapal_gpu_" + name)(None, ctypes.byref(site) if site is not None else None, *args)
    return rc, L.mapal_gpu_last_error().decode()


def with_(site, **kw):
    for k, v in kw.items():
        setattr(site, k, v)
    return site


ACCEPTED = (INVALID, "ctx is null")


def norm(site, x=P, w=P, b=P, y=2 * P, mean=P, rstd=P):
    return call("layer_norm", site, x, w, b, y, mean, rstd)


def norm_grad(site, x=P, w=P, mean=P, rstd=P, dy=2 * P, dx=3 * P, dw=P, db=P, work=P, n=1 << 30):
    return call("layer_norm_grad", site, x, w, mean, rstd, dy, dx, dw, db, work, n)


def test_layer_norm_accepts():
    for t in ("float32", "float16", "bfloat16"):
        for wt in (t, "float32"):
            assert norm(fb.norm_site(3, 5, t, wdtype=wt)) == ACCEPTED
            assert norm_grad(fb.norm_site(3, 5, t, wdtype=wt)) == ACCEPTED
    assert norm(fb.norm_site(3, 5, "float32"), w=None, b=None, mean=None, rstd=None) == ACCEPTED
    assert norm_grad(fb.norm_site(3, 5, "float32"), w=None, dw=None, db=None, work=None, n=0) == ACCEPTED
    assert norm(fb.norm_site(0, 5, "float32"), x=None, y=None) == (0, fb.lib().mapal_gpu_last_error().decode())


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "f32, f16 or bf16"), (dict(dtype=9), "f32, f16 or bf16"), (dict(dtype=-1), "f32, f16 or bf16"),
    (dict(dtype=2, wtype=1), "weight's type"), (dict(d=0), "elements"), (dict(d=1 << 31), "elements"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(ldx=4), "stride"), (dict(ldx=1 << 61), "stride"),
])
def test_layer_norm_refuses_record(change, text):
    for f in (norm, norm_grad):
        rc, msg = f(with_(fb.norm_site(3, 5, "float32"), **change))
        assert rc == INVALID and text in msg, msg


def test_layer_norm_refuses_pointers():
    s = fb.norm_site(3, 5, "float32")
    assert norm(None)[0] == INVALID
    for kw in (dict(x=None), dict(y=None)):
        assert norm(s, **kw) == (INVALID, "null x or y")
    for kw in (dict(x=P + 2), dict(y=P + 1), dict(w=P + 2), dict(b=P + 2), dict(mean=P + 1), dict(rstd=P + 2)):
        assert "not aligned" in norm(s, **kw)[1]
    assert "stride" in norm(with_(fb.norm_site(3, 5, "float32"), ldy=4))[1]
    for kw in (dict(x=None), dict(mean=None), dict(rstd=None), dict(dy=None), dict(dx=None)):
        assert "null" in norm_grad(s, **kw)[1]
    for kw in (dict(work=None), dict(work=P + 8)):
        assert "work" in norm_grad(s, **kw)[1]
    for kw in (dict(dw=P + 2), dict(db=P + 2), dict(dy=P + 2)):
        assert "not aligned" in norm_grad(s, **kw)[1]
    for kw in (dict(lddy=4), dict(lddx=4)):
        assert "stride" in norm_grad(with_(fb.norm_site(3, 5, "float32"), **kw))[1]
    assert "same stride" in norm(with_(fb.norm_site(3, 5, "float32"), ldy=6), x=P, y=P)[1]
    assert norm(with_(fb.norm_site(3, 5, "float32"), ldy=5), x=P, y=P) == ACCEPTED
    assert "same stride" in norm_grad(with_(fb.norm_site(3, 5, "float32"), lddx=6), x=2 * P, dy=P, dx=P)[1]
    assert norm_grad(s, x=2 * P, dy=P, dx=P) == ACCEPTED
    assert "same stride" in norm_grad(with_(fb.norm_site(3, 5, "float32"), lddx=6), x=P, dy=2 * P, dx=P)[1]
    # one row has no stride
    assert norm(with_(fb.norm_site(1, 5, "float32"), ldx=0, ldy=0)) == ACCEPTED
    assert call("layer_norm_grad_workspace", s, None) == (INVALID, "bytes is null")


def experts(**kw):
    return with_(fb.expert_site(6, 2, 4, 5, "float32"), **kw)


def test_experts_accept():
    assert call("expert_sort", experts(), P, P, P, P) == ACCEPTED
    assert call("expert_sort", experts(), P, P, None, P) == ACCEPTED
    assert call("expert_sort", experts(tokens=0), None, P, None, None) == ACCEPTED  # offsets are still written
    assert call("expert_dispatch", experts(), P, None, P, P, None) == ACCEPTED
    assert call("expert_dispatch", experts(dtype=3), P + 1, P, P, P + 1, P) == ACCEPTED
    assert call("expert_combine", experts(), P, None, P, P) == ACCEPTED
    assert call("expert_dispatch_grad", experts(), P, P, P) == ACCEPTED
    assert call("expert_combine_grad", experts(), P, None, P, P, P, None) == ACCEPTED


@pytest.mark.parametrize("change,rc,text", [
    (dict(k=0), INVALID, "k is 0"), (dict(experts=0), INVALID, "experts is 0"), (dict(experts=1025), UNSUPPORTED, "1024"),
    (dict(tokens=1 << 30), INVALID, "2^31"), (dict(tokens=1 << 63), INVALID, "2^31"),
])
def test_experts_refuse_record(change, rc, text):
    for name, n in (("expert_sort", 4), ("expert_dispatch", 5), ("expert_combine", 4), ("expert_dispatch_grad", 3),
                    ("expert_combine_grad", 6)):
        got, msg = call(name, experts(**change), *[P] * n)
        assert got == rc and text in msg, (name, msg)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=7), "type"), (dict(rows=1 << 31), "sorted rows"), (dict(d=1 << 31, ldt=1 << 31, ldr=1 << 31), "2^31 elements"), (dict(ldt=4), "stride"), (dict(ldr=4), "stride"),
    (dict(ldt=1 << 61), "stride"),
])
def test_expert_rows_refuse_record(change, text):
    for name, n in (("expert_dispatch", 5), ("expert_combine", 4), ("expert_dispatch_grad", 3),
                    ("expert_combine_grad", 6)):
        got, msg = call(name, experts(**change), *[P] * n)
        assert got == INVALID and text in msg, (name, msg)


def test_experts_refuse_pointers():
    for args in ((None, P, P, P), (P, None, P, P), (P, P, P, None)):
        assert "null" in call("expert_sort", experts(), *args)[1]
    for args in ((P + 2, P, P, P), (P, P + 1, P, P), (P, P, P + 2, P), (P, P, P, P + 3)):
        assert "not aligned" in call("expert_sort", experts(), *args)[1]
    for args in ((None, None, P, P, None), (P, None, None, P, None), (P, None, P, None, None)):
        assert "null" in call("expert_dispatch", experts(), *args)[1]
    for args in ((P, P, P, P, None), (P, None, P, P, P)):
        assert "come together" in call("expert_dispatch", experts(), *args)[1]
    assert "not aligned" in call("expert_dispatch", experts(), P + 2, None, P, P, None)[1]
    for args in ((None, P, P, P), (P, P, None, P), (P, P, P, None)):
        assert "null" in call("expert_combine", experts(), *args)[1]
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert "null" in call("expert_dispatch_grad", experts(), *args)[1]
    for args in ((None, P, P, P, P, P), (P, P, None, P, P, P), (P, P, P, None, P, P), (P, P, P, P, None, P)):
        assert "null" in call("expert_combine_grad", experts(), *args)[1]
    # 8-bit rows are moved, not summed
    for name, n in (("expert_combine", 4), ("expert_dispatch_grad", 3), ("expert_combine_grad", 6)):
        assert "type" in call(name, experts(dtype=3), *[P] * n)[1]


def quant(**kw):
    return with_(fb.quant_site(3, 5, "bfloat16"), **kw)


def test_quantize_refusals():
    assert call("quantize_rows_i8", quant(), P, P + 1, P) == ACCEPTED
    assert call("quantize_rows_i8", quant(d=0, ldx=0, ldq=0), None, None, P) == ACCEPTED  # scales of nothing: 0
    for kw, text in ((dict(dtype=3), "f32, f16"), (dict(dtype=5), "f32, f16"), (dict(ldx=4), "stride"),
                     (dict(ldq=4), "stride"), (dict(d=1 << 31), "stride")):
        rc, msg = call("quantize_rows_i8", quant(**kw), P, P, P)
        assert rc == INVALID and text in msg
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert "null" in call("quantize_rows_i8", quant(), *args)[1]
    for args in ((P + 1, P, P), (P, P, P + 2)):
        assert "not aligned" in call("quantize_rows_i8", quant(), *args)[1]


def mm(**kw):
    return with_(fb.matmul_i8_site(3, 4, 5, "float32"), **kw)


def test_matmul_i8_refusals():
    assert call("matmul_i8", mm(), P + 1, P, P + 3, P, None, P) == ACCEPTED
    assert call("matmul_i8", mm(), P, None, P, None, P, P) == ACCEPTED
    assert call("matmul_i8", mm(k=0), None, P, None, P, None, P) == ACCEPTED
    assert call("matmul_i8", with_(fb.matmul_i8_site(3, 4, 5, "bfloat16", groups=7)), P, P, P, P, P, P) == ACCEPTED
    assert call("matmul_i8", mm(m=0), None, None, None, None, None, None)[0] == 0
    for kw, rc, text in ((dict(dtype=3), INVALID, "C is f32"), (dict(groups=0), INVALID, "groups"),
                         (dict(groups=1 << 17), INVALID, "groups"), (dict(k=131072, lda=131072, ldb=131072), UNSUPPORTED, "32 bits"),
                         (dict(m=1 << 31), UNSUPPORTED, "2^31"), (dict(n=1 << 31, ldc=1 << 31), UNSUPPORTED, "2^31"),
                         (dict(m=0x7fffff01), UNSUPPORTED, "2^31"),
                         (dict(lda=4), INVALID, "stride"), (dict(ldb=4), INVALID, "stride"), (dict(ldc=3), INVALID, "stride"),
                         (dict(groups=2, ldg=19), INVALID, "between groups")):
        got, msg = call("matmul_i8", mm(**kw), P, P, P, P, P, P)
        assert got == rc and text in msg, msg
    assert "need offsets" in call("matmul_i8", mm(groups=2), P, P, P, P, None, P)[1]
    for args in ((None, P, P, P, None, P), (P, P, None, P, None, P), (P, P, P, P, None, None)):
        assert "null" in call("matmul_i8", mm(), *args)[1]
    for args in ((P, P + 1, P, P, None, P), (P, P, P, P + 2, None, P), (P, P, P, P, P + 2, P), (P, P, P, P, None, P + 2)):
        assert "not aligned" in call("matmul_i8", mm(), *args)[1]


# ---- the wrappers' checks ----------------------------------------------------------------------


@pytest.fixture
def ctx():
    c = fb.Context.__new__(fb.Context)
    c._h, c.devices = None, [-1]  # the device number of a CPU tensor; the call itself then ends with "ctx is null"
    return c


def test_wrapper_passes_good_tensors_on(ctx):
    x = torch.zeros(3, 8)[:, :5]
    w, y = torch.zeros(5), torch.zeros(3, 5)
    with pytest.raises(fb.MapalInfraError, match="ctx is null"):
        ctx.layer_norm(fb.norm_site(3, 5, x.dtype, ldx=8), x, w, w, y)
    with pytest.raises(fb.MapalInfraError, match="ctx is null"):
        ctx.layer_norm(fb.norm_site(3, 5, x.dtype, ldx=8), x.data_ptr(), None, None, y.reshape(-1))


@pytest.mark.parametrize("site,x,text", [
    (dict(), torch.zeros(3, 5, dtype=torch.bfloat16), "the record says"),
    (dict(), torch.zeros(2, 5), "holds 10 elements"),
    (dict(), torch.zeros(1).expand(3, 5), "contiguous"),
    (dict(ldx=8), torch.zeros(3, 5), "row stride 5"),
    (dict(ldx=8), torch.zeros(15), "holds 15 elements"),
    (dict(ldx=8), torch.zeros(3, 9)[:, :5], "row stride 9"),
    (dict(), torch.zeros(5, 3).t(), "contiguous"),
])
def test_wrapper_refuses(ctx, site, x, text):
    w, y = torch.zeros(5), torch.zeros(3, 5)
    with pytest.raises(ValueError, match=text):
        ctx.layer_norm(fb.norm_site(3, 5, "float32", **site), x, w, w, y)


def test_wrapper_refuses_other_arguments(ctx):
    i, f, b = torch.zeros(12, dtype=torch.int32), torch.zeros(12), torch.zeros(3, 5, dtype=torch.int8)
    e = fb.expert_site(6, 2, 4, 5, "float32")
    with pytest.raises(ValueError, match="ids is torch.int64"):
        ctx.expert_sort(e, i.long(), i, i, i)
    with pytest.raises(ValueError, match="offsets holds 4"):
        ctx.expert_sort(e, i, i[:4].clone(), i, i)
    with pytest.raises(ValueError, match="xs holds 20"):
        ctx.expert_dispatch(e, torch.zeros(6, 5), i, torch.zeros(4, 5))
    with pytest.raises(ValueError, match="w is torch.bfloat16"):
        ctx.expert_combine(e, torch.zeros(12, 5), f.bfloat16(), i, torch.zeros(6, 5))
    with pytest.raises(ValueError, match="dw holds 3"):
        ctx.expert_combine_grad(e, torch.zeros(12, 5), f, i, torch.zeros(6, 5), torch.zeros(12, 5), f[:3].clone())
    with pytest.raises(ValueError, match="q is torch.uint8"):
        ctx.quantize_rows_i8(fb.quant_site(3, 5, "float32"), torch.zeros(3, 5), b.to(torch.uint8), f)
    with pytest.raises(ValueError, match="B holds 15"):
        ctx.matmul_i8(fb.matmul_i8_site(3, 3, 5, "float32", groups=2), b, f, b, f, f, offsets=i)
    ctx.devices = [0]
    with pytest.raises(ValueError, match="ids is on cpu"):
        ctx.expert_sort(e, i, i, i, i)
    with pytest.raises(ValueError, match="work is on cpu"):
        ctx.layer_norm_grad(fb.norm_site(3, 4, "float32"), 64, None, 64, 64, 64, 64, 64, 64, torch.zeros(9))
    with pytest.raises(ValueError, match="no element type"):
        fb.norm_site(3, 5, torch.float64)


BATCH = torch.zeros(4, 6, 5)  # 4 sequences of 6 tokens


@pytest.mark.parametrize("x,rows,ld,text", [
    (BATCH[:, :3], 12, 0, "stride 30 in dimension 0, the record says 15"),  # a padded batch is not evenly spaced rows
    (BATCH[:, :, :4], 24, 5, None), (BATCH[1:, :, :4], 18, 5, None), (BATCH[:, 2], 4, 30, None),
    (BATCH[:, 2], 4, 0, "row stride 30"), (BATCH[:, 2:3], 4, 30, None), (BATCH[:, 2:3], 4, 5, "row stride 30"),
    (BATCH[::2], 12, 0, "stride 60 in dimension 0, the record says 30"), (BATCH.transpose(0, 1), 24, 0, "row stride 30"),
    (BATCH.view(4, 2, 3, 5)[:, :, :2], 16, 0, "stride 15 in dimension 1, the record says 10"),
])
def test_wrapper_takes_views_as_they_lie(ctx, x, rows, ld, text):
    d = x.shape[-1]
    site = fb.norm_site(rows, d, "float32", ldx=ld)
    with pytest.raises(ValueError if text else fb.MapalInfraError, match=text or "ctx is null"):
        ctx.layer_norm(site, x, None, None, torch.zeros(rows, d))


def test_wrapper_refuses_views_of_what_has_no_stride(ctx):
    e, x, ids = fb.expert_site(6, 2, 4, 5, "float32"), torch.zeros(6, 5), torch.zeros(12, dtype=torch.int32)
    wide = torch.zeros(6, 8, dtype=torch.int32)[:, :2]  # the first 2 of 8
    with pytest.raises(ValueError, match="ids must be contiguous"):
        ctx.expert_sort(e, wide, ids, ids, ids)
    with pytest.raises(ValueError, match="pos must be contiguous"):
        ctx.expert_dispatch(e, x, wide, torch.zeros(12, 5))
    with pytest.raises(ValueError, match="w must be contiguous"):
        ctx.expert_combine(e, torch.zeros(12, 5), torch.zeros(6, 8)[:, :2], ids, x)
    with pytest.raises(ValueError, match="scale_out must be contiguous|elements of a row"):
        ctx.expert_dispatch(e, x, ids, torch.zeros(12, 5), scale=torch.zeros(6), scale_out=torch.zeros(24)[::2])


def test_wrapper_checks_the_stride_between_matrices(ctx):
    a, f, off = torch.zeros(3, 5, dtype=torch.int8), torch.zeros(12), torch.zeros(3, dtype=torch.int32)
    b = torch.zeros(4, 3, 8, dtype=torch.int8)
    c = torch.zeros(3, 3)
    run = lambda B, **kw: ctx.matmul_i8(fb.matmul_i8_site(3, 3, 5, "float32", groups=2, **kw), a, f, B, f, c, offsets=off)
    for B, kw in ((b[:2, :, :5], dict(ldb=8, ldg=24)), (b[::2, :, :5], dict(ldb=8, ldg=48)), (b[1:3, :, 3:], dict(ldb=8))):
        with pytest.raises(fb.MapalInfraError, match="ctx is null"):
            run(B, **kw)
    with pytest.raises(ValueError, match="stride 48 in dimension 0, the record says 24"):
        run(b[::2, :, :5], ldb=8)
    with pytest.raises(ValueError, match="row stride 8"):
        run(b[:2, :, :5])


# ---- the calls without ctypes --------------------------------------------------------------------


def test_direct_calls_take_what_the_methods_take(ctx):
    """Plain tensors go through, as the refusal of the C entry shows; everything else is left to the method."""
    i, f = torch.zeros(12, dtype=torch.int32), torch.zeros(64)
    z = lambda *s: torch.zeros(*s)  # noqa: E731
    with pytest.raises(fb.MapalInfraError, match="ctx is null"):
        ctx.layer_norm(fb.norm_site(3, 5, "float32"), z(3, 5), None, None, z(3, 5))  # binds them
    D, h = fb._direct, ctypes.c_void_p()
    n, e, q = fb.norm_site(3, 5, "float32"), fb.expert_site(6, 2, 4, 5, "float32"), fb.quant_site(3, 5, "float32")
    m = fb.matmul_i8_site(3, 4, 5, "float32", groups=2)
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8)  # noqa: E731
    calls = {
        "layer_norm": (n, [z(3, 5), z(5), z(5), z(3, 5), z(3), z(3)]),
        "layer_norm_grad": (n, [z(3, 5), z(5), z(3), z(3), z(3, 5), z(3, 5), z(5), z(5), z(64)]),
        "expert_sort": (e, [i, i[:5].clone(), i, i]),
        "expert_dispatch": (e, [z(6, 5), i, z(12, 5), z(6), z(12)]),
        "expert_combine": (e, [z(12, 5), z(12), i, z(6, 5)]),
        "expert_dispatch_grad": (e, [z(12, 5), i, z(6, 5)]),
        "expert_combine_grad": (e, [z(12, 5), z(12), i, z(6, 5), z(12, 5), z(12)]),
        "quantize_rows_i8": (q, [z(3, 5), i8(3, 5), z(3)]),
        "matmul_i8": (m, [i8(3, 5), z(3), i8(2, 4, 5), z(2, 4), z(3, 4), i[:3].clone()]),
    }
    assert set(calls) == set(fb._Direct.NAMES)
    for name, (site, args) in calls.items():
        call = getattr(D, name)
        # the C entry refuses the null context, or an address that is not as aligned as CPU memory happens to be
        assert call(h, -1, site, *args) == INVALID, name
        assert "null" in fb.lib().mapal_gpu_last_error().decode() or "align" in fb.lib().mapal_gpu_last_error().decode()
        assert call(h, 0, site, *args) is None  # another device
        assert call(None, -1, site, *args) is None and call(h, -1, None, *args) is None
        assert call(h, -1, q if site is not q else n, *args) is None  # another record
        assert call(h, -1, site, *args[:-1]) is None and call() is None
        for k, t in enumerate(args):
            for bad in (t.data_ptr(), "x", t.double(), t.flatten()[:-1]):
                if name == "layer_norm_grad" and k == 8 and not isinstance(bad, (int, str)):
                    continue  # scratch of any type; its length is the entry's to check
                assert call(h, -1, site, *args[:k], bad, *args[k + 1:]) is None, (name, k)
            wide = torch.stack([t, t], -1)[..., 0]  # every second element
            if t.numel() > 1:
                assert call(h, -1, site, *args[:k], wide, *args[k + 1:]) is None, (name, k)
    # matrices at the record's stride go through, others are left to the method
    s = fb.norm_site(3, 5, "float32", ldx=8, ldy=7)
    x, y = torch.zeros(3, 8), torch.zeros(3, 7)
    for a, b, ok in ((x[:, :5], y[:, 1:6], True), (x[:, 1:6], y[:, 2:], True), (x[:, :5], z(3, 9)[:, :5], False),
                     (x[:, :5].t(), y[:, :5], False), (x[:2, :5], y[:, :5], True), (x[1:, :5], y[:, :5], False),
                     (x[:1, :5], y[:, :5], False), (x.view(3, 2, 4)[:, :, :3], y[:, :5], False)):
        assert (D.layer_norm(h, -1, s, a, None, None, b, None, None) is not None) is ok
    # the record is read on every call
    n.rows = 4
    assert D.layer_norm(h, -1, n, *calls["layer_norm"][1]) is None
    n.rows, n.d = 1, 4
    assert D.layer_norm(h, -1, n, *calls["layer_norm"][1]) == INVALID

"""The loss of a large vocabulary and its gradients on a B200, against the formula in f64.

Bounds: a logit is a sum of d exact products on the tensor cores, d/16 steps of 17 terms, each cut at one unit in
the last place: err_l <= (d + 16)*17/16*2*U32 * sum |h||w| (as in test_gpu_product.py). The exponent l*log2(e) - m*log2(e)
is rounded twice, ex2 is off by 2^-22 at most and sums of V terms in chunks by 2^-19 (32 terms a chunk, 4 chains, and
the joins): relative errors of a sum of exponentials, so absolute ones of its logarithm."""
import pytest
import torch

import flow_b200 as fb
from _rows import U32, Guarded, assert_within, half_step, out_error, replayed

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def inputs(rows, vocab, d, dtype, seed, ignored=0.0, sure=0.0, pads=(0, 0), offsets=(0, 0), scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    w = Guarded(vocab, d, dtype, pads[1], offsets[1]).put(r(vocab, d) / d ** 0.5 * scale)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    h = Guarded(rows, d, dtype, pads[0], offsets[0]).put(r(rows, d) + sure * w.t[t].float())
    if ignored:
        t[torch.rand(rows, generator=g, device="cuda") < ignored] = -1
    dloss = torch.rand(rows, generator=g, device="cuda") + 0.1
    return h, w, t.to(torch.int32), dloss


def formula(h, w, t, dloss, dtype):
    """loss, lse, dh, dw in f64 and bounds on each."""
    h, w, there = h.double(), w.double(), t >= 0
    h = torch.where(there[:, None], h, 0.0)
    at = t.long().clamp(min=0)[:, None]
    l, size = h @ w.t(), h.abs() @ w.abs().t()
    d, v = h.shape[1], w.shape[0]
    err_l = (d + 16) * 17 / 16 * 2 * U32 * size
    lse = torch.logsumexp(l, 1)
    lse32 = torch.where(there, lse, 0.0).float()
    loss = lse - l.gather(1, at)[:, 0]
    big = l.abs().amax(1)
    expo = 4 * U32 * 1.4427 * 2 * big + 2.0 ** -22 + 2.0 ** -19  # of a sum of exponentials, relative
    err_lse = err_l.amax(1) + expo + 8 * U32 * big
    err_loss = 2 * err_l.amax(1) + expo + 8 * U32 * (big + loss)
    z = torch.zeros_like(loss)
    p = torch.exp(l - lse32.double()[:, None])
    g = torch.where(there, dloss.double(), 0.0)[:, None]
    dl = p.clone()
    dl.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    dl *= g
    # p carries its logit's and lse's errors, dl one rounding to the rows' type (f16: also a step of 2^-24 at the scale
    # that brings the largest gradient to 2^14 or more)
    err_dl = g * (p * (err_l + 4 * U32 * 1.4427 * (l.abs() + lse32.double().abs()[:, None]) + 2.0 ** -21) + 2 * U32)
    err_dl += (dl.abs() + err_dl) * half_step(dtype) + (g.max() * 2.0 ** -38 if dtype == torch.float16 else 0.0)
    dh, dw = dl @ w, dl.t() @ h
    steps = 17 / 16 * 2 * U32
    pieces = 8 * U32  # sums of pieces in f32
    err_dh = err_dl @ w.abs() + ((v + 16) * steps + pieces) * ((dl.abs() + err_dl) @ w.abs())
    err_dw = err_dl.t() @ h.abs() + ((h.shape[0] + 16) * steps + pieces) * ((dl.abs() + err_dl).t() @ h.abs())
    err_dh += out_error(dh.abs() + err_dh, dtype)
    err_dw += out_error(dw.abs() + err_dw, dtype)
    return ((torch.where(there, loss, z), torch.where(there, err_loss, z)),
            (torch.where(there, lse, z), torch.where(there, err_lse, z)), (dh, err_dh), (dw, err_dw)), lse32


def check(ctx, h, w, t, dloss, opads=(0, 0), call=lambda f: f()):
    rows, d = h.t.shape
    vocab, dtype = w.t.shape[0], h.t.dtype
    want, lse32 = formula(h.t, w.t, t, dloss, dtype)
    dh, dw = Guarded(rows, d, dtype, opads[0], opads[0]), Guarded(vocab, d, dtype, opads[1], opads[1])
    site = fb.loss_site(rows, vocab, d, dtype, ldh=h.ld, ldw=w.ld, lddh=dh.ld, lddw=dw.ld)
    n = ctx.linear_loss_workspace(site, w=w.t)
    buf = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    loss, lse = (torch.full((rows + 1,), 9.0, device="cuda") for _ in range(2))

    def go():
        ctx.linear_loss(site, h.t, w.t, t, loss, lse, buf[:n])
        ctx.linear_loss_grad(site, h.t, w.t, t, lse32, dloss, dh.t, dw.t, buf[:n])

    call(go)
    for got, (value, bound), what in zip((loss[:rows], lse[:rows], dh.t, dw.t), want, ("loss", "lse", "dh", "dw")):
        assert_within(got, value, bound, what)
    assert (loss[rows] == 9.0) and (lse[rows] == 9.0) and dh.intact() and dw.intact()
    assert (buf[n:] == 0xA5).all(), "written behind work"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,vocab,d", [(1, 1, 1), (1, 2, 8), (3, 5, 7), (1, 1000, 64), (7, 129, 40), (33, 257, 100), (64, 4096, 72),
                                          (129, 1003, 65), (256, 256, 128), (300, 2500, 96), (1000, 300, 264), (2, 9000, 512),
                                          (513, 1025, 24), (50, 128, 1100)])
def test_sizes(ctx, rows, vocab, d, dtype):
    check(ctx, *inputs(rows, vocab, d, dtype, rows + vocab + d))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("ignored", [0.1, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("rows,vocab,d", [(40, 300, 64), (700, 1000, 136), (2000, 515, 33)])
def test_rows_without_a_target(ctx, rows, vocab, d, ignored, dtype):
    check(ctx, *inputs(rows, vocab, d, dtype, rows, ignored))


@pytest.mark.parametrize("pads,offsets,opads", [((8, 8), (0, 0), (8, 16)), ((1, 0), (0, 0), (1, 3)), ((0, 5), (0, 0), (0, 0)),
                                                ((8, 8), (1, 0), (0, 0)), ((8, 8), (0, 3), (2, 0)), ((16, 24), (8, 16), (3, 5))])
@pytest.mark.parametrize("rows,vocab,d", [(70, 600, 72), (300, 1300, 131)])
def test_strides_and_places(ctx, rows, vocab, d, pads, offsets, opads):
    check(ctx, *inputs(rows, vocab, d, torch.bfloat16, 5, 0.2, pads=pads, offsets=offsets), opads=opads)


@pytest.mark.parametrize("dtype", HALF)
def test_several_pieces(ctx, dtype):
    """Rows enough that the vocabulary is taken in several pieces: dh is summed over them."""
    h, w, t, dloss = inputs(9000, 33000, 72, dtype, 3, 0.05)
    check(ctx, h, w, t, dloss)


def test_several_pieces_of_copied_weights(ctx):
    check(ctx, *inputs(300, 70001, 2051, torch.bfloat16, 3))


@pytest.mark.parametrize("dtype", HALF)
def test_small_gradients(ctx, dtype):
    """The gradients of a mean over many rows, and rows whose share is far below the others'."""
    h, w, t, dloss = inputs(200, 3000, 64, dtype, 4)
    check(ctx, h, w, t, dloss / 1e6 if dtype == torch.bfloat16 else dloss / 256)
    check(ctx, h, w, t, torch.where(torch.arange(200, device="cuda") % 3 == 0, dloss, dloss / 1024))
    check(ctx, h, w, t, torch.zeros_like(dloss))


def test_negative_and_no_loss_gradient(ctx):
    h, w, t, dloss = inputs(100, 500, 64, torch.bfloat16, 6)
    check(ctx, h, w, t, torch.where(torch.arange(100, device="cuda") % 2 == 0, dloss, torch.zeros_like(dloss)))
    site = fb.loss_site(100, 500, 64, torch.bfloat16)
    work = torch.empty(ctx.linear_loss_workspace(site), dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(100, device="cuda") for _ in range(2))
    ctx.linear_loss(site, h.t, w.t, t, loss, lse, work)
    a, b = (torch.empty(100, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ctx.linear_loss_grad(site, h.t, w.t, t, lse, None, a, None, work)
    ctx.linear_loss_grad(site, h.t, w.t, t, lse, torch.ones(100, device="cuda"), b, None, work)
    assert torch.equal(a, b)
    ctx.linear_loss_grad(site, h.t, w.t, t, lse, -torch.ones(100, device="cuda"), b, None, work)
    assert torch.equal(a, -b)


@pytest.mark.parametrize("dtype", HALF)
def test_nearly_certain_targets(ctx, dtype):
    """Where the target takes nearly everything the loss is the others' share: its own relative error is small. Here h
    is 12 or more times the target's weights, whole sixteenths, so that every logit is exact in f32."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, vocab, d = 50, 700, 64
    w = (torch.randint(-8, 9, (vocab, d), generator=g, device="cuda") / 16.0).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    h = (w[t].float() * torch.randint(2, 5, (rows, 1), generator=g, device="cuda")).to(dtype)
    site = fb.loss_site(rows, vocab, d, dtype)
    work = torch.empty(ctx.linear_loss_workspace(site, grad=False), dtype=torch.uint8, device="cuda")
    loss = torch.empty(rows, device="cuda")
    ctx.linear_loss(site, h, w, t.to(torch.int32), loss, None, work)
    l = h.double() @ w.double().t()
    lt = l.gather(1, t[:, None])
    others = torch.exp(l - lt).scatter(1, t[:, None], 0.0).sum(1)
    want = torch.log1p(others)
    assert want.min() < 1e-4
    assert_within(loss, want, want * (2.0 ** -18 + 16 * U32 * l.abs().amax(1)))


def test_what_rows_without_a_target_hold_is_not_read(ctx):
    h, w, t, dloss = inputs(300, 500, 64, torch.bfloat16, 7, 0.4)
    out = []
    for bad in (0.0, float("nan"), float("inf")):
        h.t[t == -1] = bad
        d2 = torch.where(t == -1, bad, dloss)
        site = fb.loss_site(300, 500, 64, torch.bfloat16)
        work = torch.full((ctx.linear_loss_workspace(site),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN
        loss, lse = (torch.empty(300, device="cuda") for _ in range(2))
        dh, dw = torch.empty(300, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(500, 64, dtype=torch.bfloat16, device="cuda")
        ctx.linear_loss(site, h.t, w.t, t, loss, lse, work)
        work.fill_(0xFF)
        ctx.linear_loss_grad(site, h.t, w.t, t, torch.where(t == -1, bad, lse), d2, dh, dw, work)
        out.append((loss, lse, dh, dw))
    for o in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], o))
    assert torch.isfinite(out[0][3]).all() and not out[0][2][t == -1].any()


@pytest.mark.parametrize("bad", [-2, 500, 1 << 30, -(1 << 31)])
def test_bad_targets_trap(ctx, bad):
    """The call traps, and the row counts as one without a target."""
    h, w, t, dloss = inputs(100, 500, 64, torch.float16, 8)
    site = fb.loss_site(100, 500, 64, torch.float16)
    work = torch.empty(ctx.linear_loss_workspace(site), dtype=torch.uint8, device="cuda")
    outs = []
    for v in (-1, bad):
        t2 = t.clone()
        t2[17] = v
        loss, lse = (torch.full((100,), 5.0, device="cuda") for _ in range(2))
        dh, dw = torch.ones(100, 64, dtype=torch.float16, device="cuda"), torch.ones(500, 64, dtype=torch.float16, device="cuda")
        for f in (lambda: ctx.linear_loss(site, h.t, w.t, t2, loss, lse, work),
                  lambda: ctx.linear_loss_grad(site, h.t, w.t, t2, lse, dloss, dh, dw, work)):
            if v == -1:
                f()
            else:
                with pytest.raises(fb.MapalTrap, match="index_oob"):
                    f()
        outs.append((loss, lse, dh, dw))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_no_rows(ctx):
    site = fb.loss_site(0, 300, 40, torch.bfloat16, lddw=48)
    z = torch.zeros(0, 40, dtype=torch.bfloat16, device="cuda")
    dw = Guarded(300, 40, torch.bfloat16, 8)
    dw.t.fill_(3)
    work = torch.empty(max(1, ctx.linear_loss_workspace(site)), dtype=torch.uint8, device="cuda")
    e = torch.zeros(0, device="cuda")
    ctx.linear_loss(site, z, torch.zeros(300, 40, dtype=torch.bfloat16, device="cuda"), e.int(), e, e, work)
    ctx.linear_loss_grad(site, z, None, e.int(), e, e, z, dw.t, work)
    assert not dw.t.any() and dw.intact()


def test_short_work_is_refused(ctx):
    h, w, t, dloss = inputs(100, 500, 64, torch.bfloat16, 9, offsets=(0, 1), pads=(0, 0))
    site = fb.loss_site(100, 500, 64, torch.bfloat16)
    loss = torch.empty(100, device="cuda")
    less, more = ctx.linear_loss_workspace(site, grad=False), ctx.linear_loss_workspace(site, w=w.t, grad=False)
    assert less < more
    with pytest.raises(fb.MapalInfraError, match="work is shorter"):
        ctx.linear_loss(site, h.t, w.t, t, loss, None, torch.empty(less, dtype=torch.uint8, device="cuda"))
    with pytest.raises(fb.MapalInfraError, match="work is shorter"):
        ctx.linear_loss(site, h.t, w.t.clone(), t, loss, None, torch.empty(less - 1, dtype=torch.uint8, device="cuda"))


def test_captured(ctx):
    h, w, t, dloss = inputs(500, 1200, 104, torch.float16, 10, 0.3)
    check(ctx, h, w, t, dloss, call=lambda f: replayed(ctx, f))


def test_differences(ctx):
    """The gradient against central differences of the f64 loss along a direction."""
    h, w, t, dloss = inputs(60, 400, 64, torch.bfloat16, 11, 0.1)
    site = fb.loss_site(60, 400, 64, torch.bfloat16)
    work = torch.empty(ctx.linear_loss_workspace(site), dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(60, device="cuda") for _ in range(2))
    dh, dw = torch.empty(60, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(400, 64, dtype=torch.bfloat16, device="cuda")
    ctx.linear_loss(site, h.t, w.t, t, loss, lse, work)
    ctx.linear_loss_grad(site, h.t, w.t, t, lse, dloss, dh, dw, work)
    g = torch.Generator(device="cuda").manual_seed(2)
    vh, vw = (torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64) for x in (dh, dw))
    there = t >= 0

    def total(e):
        l = (h.t.double() + e * vh) @ (w.t.double() + e * vw).t()
        per = torch.logsumexp(l, 1) - l.gather(1, t.long().clamp(min=0)[:, None])[:, 0]
        return (torch.where(there, per, 0.0) * dloss.double()).sum()

    e = 1e-5
    want = (total(e) - total(-e)) / (2 * e)
    got = (dh.double() * vh).sum() + (dw.double() * vw).sum()
    # each gradient is off by its bound; errors of random sign against a random direction
    (_, _, (_, eh), (_, ew)), _ = formula(h.t, w.t, t, dloss, torch.bfloat16)
    assert (got - want).abs() <= (eh * vh.abs()).sum() + (ew * vw.abs()).sum() + 1e-6 * want.abs()


def test_two_streams():
    ctxs, streams = [fb.Context((0,), sync=False) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    h, w, t, dloss = inputs(400, 2000, 128, torch.bfloat16, 12, 0.2)
    site = fb.loss_site(400, 2000, 128, torch.bfloat16)
    e = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    outs = [(e(400, dtype=torch.float32), e(400, dtype=torch.float32), e(400, 128), e(2000, 128),
             e(ctxs[0].linear_loss_workspace(site), dtype=torch.uint8)) for _ in ctxs]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s, (loss, lse, dh, dw, work) in zip(ctxs, streams, outs):
            c.set_stream(s.cuda_stream)
            c.linear_loss(site, h.t, w.t, t, loss, lse, work)
            c.linear_loss_grad(site, h.t, w.t, t, lse, dloss, dh, dw, work)
    for c in ctxs:
        c.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0][:4], outs[1][:4]))
    want, _ = formula(h.t, w.t, t, dloss, torch.bfloat16)
    assert_within(outs[0][0], *want[0])
    for c in ctxs:
        c.close()


def test_the_mean_cut_of_the_sums_is_given_back(ctx):
    """The tensor cores cut a sum at each step of 16 products: d/16 * 2^-26 of a logit in the mean. lse, an average of
    logits, would be that much of their average too small for every row; at most a quarter of it is left in the mean."""
    rows, vocab, d = 256, 20000, 2048
    g = torch.Generator(device="cuda").manual_seed(13)
    w = (torch.randn(vocab, d, generator=g, device="cuda") * (1.5 / d ** 0.5)).to(torch.bfloat16)
    h = torch.randn(rows, d, generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    site = fb.loss_site(rows, vocab, d, torch.bfloat16)
    work = torch.empty(ctx.linear_loss_workspace(site, grad=False), dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(rows, device="cuda") for _ in range(2))
    ctx.linear_loss(site, h, w, t, loss, lse, work)
    l = h.double() @ w.double().t()
    want = torch.logsumexp(l, 1)
    average = (torch.softmax(l, 1) * l).sum(1).mean()
    assert (lse.double() - want).mean().abs() <= 0.25 * d / 16 * 2.0 ** -26 * average

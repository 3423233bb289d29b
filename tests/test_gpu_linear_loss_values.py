"""The loss of a large vocabulary on a B200 where its values could go wrong: the log-sum of rows without a target."""
import pytest
import torch

import flow_b200 as fb
from _rows import U32, Guarded, assert_within, half_step, out_error, replayed
from test_gpu_linear_loss import HALF, formula, inputs
from test_gpu_training_step import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def sums(h, w, t):
    """lse of every row, the loss (0 without a target) in f64, and bounds on both: a logit's, of the exponentials and
    of their sum as in test_gpu_linear_loss.py."""
    h, w, there = h.double(), w.double(), t >= 0
    l, size = h @ w.t(), h.abs() @ w.abs().t()
    err_l = ((h.shape[1] + 16) * 17 / 16 * 2 * U32 * size).amax(1)
    big = l.abs().amax(1)
    lse = torch.logsumexp(l, 1)
    loss = torch.where(there, lse - l.gather(1, t.long().clamp(min=0)[:, None])[:, 0], 0.0)
    err = err_l + 8 * U32 * big * (1 + 1.4427) + 2.0 ** -22 + 2.0 ** -19
    return (lse, err), (loss, torch.where(there, err + err_l + 8 * U32 * loss, 0.0))


def forward(ctx, h, w, t, ask=True, call=lambda f: f()):
    rows, d = h.t.shape
    site = fb.loss_site(rows, w.t.shape[0], d, h.t.dtype, ldh=h.ld, ldw=w.ld)
    work = torch.full((ctx.linear_loss_workspace(site, w=w.t, grad=False),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN
    loss, lse = (torch.full((rows,), 9.0, device="cuda") for _ in range(2))
    call(lambda: ctx.linear_loss(site, h.t, w.t, t, loss, lse if ask else None, work))
    return loss, lse


def check(ctx, h, w, t, dloss, opads=(0, 0), call=lambda f: f(), at=0):
    """The loss, every row's lse and both gradients, with nothing written around them or around work, which begins `at`
    bytes behind a boundary of 256."""
    (rows, d), (vocab, dtype) = h.t.shape, (w.t.shape[0], h.t.dtype)
    (_, _, *want), lse32 = formula(h.t, w.t, t, dloss, dtype)
    lse_loss = sums(h.t, w.t, t)
    dh, dw = Guarded(rows, d, dtype, opads[0], opads[0]), Guarded(vocab, d, dtype, opads[1], opads[1])
    site = fb.loss_site(rows, vocab, d, dtype, ldh=h.ld, ldw=w.ld, lddh=dh.ld, lddw=dw.ld)
    n = ctx.linear_loss_workspace(site, w=w.t)
    buf = torch.full((at + n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    work = buf[at:at + n]
    lse, loss = (torch.full((rows + 1,), 9.0, device="cuda") for _ in range(2))

    def go():
        ctx.linear_loss(site, h.t, w.t, t, loss, lse, work)
        ctx.linear_loss_grad(site, h.t, w.t, t, lse32, dloss, dh.t, dw.t, work)

    call(go)
    for got, (value, bound), what in zip((lse[:rows], loss[:rows], dh.t, dw.t), (*lse_loss, *want), ("lse", "loss", "dh", "dw")):
        assert_within(got, value, bound, what)
    assert (loss[rows] == 9.0) and (lse[rows] == 9.0) and dh.intact() and dw.intact() and (buf[:at] == 0xA5).all() and (buf[at + n:] == 0xA5).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("ignored", [0.0, 0.1, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("rows,vocab,d", [(40, 300, 64), (700, 1000, 136), (2000, 515, 33)])
def test_gradients_beside_rows_without_a_target(ctx, rows, vocab, d, ignored, dtype):
    check(ctx, *inputs(rows, vocab, d, dtype, rows, ignored))


@pytest.mark.parametrize("pads,offsets,opads", [((8, 8), (0, 0), (8, 16)), ((1, 0), (0, 0), (1, 3)), ((0, 5), (0, 0), (0, 0)),
                                                ((8, 8), (1, 0), (0, 0)), ((8, 8), (0, 3), (2, 0)), ((16, 24), (8, 16), (3, 5))])
@pytest.mark.parametrize("rows,vocab,d", [(70, 600, 72), (300, 1300, 131)])
def test_strides_and_places(ctx, rows, vocab, d, pads, offsets, opads):
    check(ctx, *inputs(rows, vocab, d, torch.float16, 5, 0.2, pads=pads, offsets=offsets), opads=opads)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("at", [16, 32, 48, 128, 240])
@pytest.mark.parametrize("rows,vocab,d,offset", [(40, 300, 64, 0), (700, 1000, 136, 0), (300, 600, 33, 1)])
def test_scratch_on_any_16_bytes(ctx, rows, vocab, d, offset, at, dtype):
    """As a slice of an arena lies: on 16 bytes, whatever lies on 32 of its own."""
    check(ctx, *inputs(rows, vocab, d, dtype, rows, 0.2, offsets=(0, offset)), at=at)


def test_several_pieces_and_captured(ctx):
    check(ctx, *inputs(9000, 33000, 72, torch.bfloat16, 3, 0.05), call=lambda f: replayed(ctx, f))


def test_the_loss_of_a_training_step(ctx):
    """On what a step of a layer of experts gave it, forty rows of padding among its rows."""
    s = Step()
    s.run(ctx)
    (lse, elses), (loss, eloss) = sums(s.out, s.wv, s.targets)
    assert_within(s.lse, lse, elses, "lse")
    assert_within(s.loss, loss, eloss, "loss")
    (_, _, (dh, edh), (dw, edw)), _ = formula(s.out, s.wv, s.targets, s.g, s.t)
    # the step's own lse goes into its gradient: its error is a relative one of p
    assert_within(s.dout, dh, edh + 2 * elses.max() * (s.g.max() * s.wv.double().abs().sum(0)), "dh")
    assert_within(s.dwv, dw, edw + 2 * elses.max() * (s.g.double() @ s.out.double().abs()), "dw")
    assert not s.dout[s.T - 40:].any() and torch.isfinite(s.dx.float()).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("ignored", [0.0, 0.1, 0.97, 1.0])
@pytest.mark.parametrize("rows,vocab,d,pads,offsets", [(1, 1, 1, (0, 0), (0, 0)), (1, 300, 64, (0, 0), (0, 0)),
                                                       (40, 129, 7, (1, 0), (0, 3)), (700, 1000, 136, (8, 16), (0, 0)),
                                                       (2500, 515, 33, (0, 0), (1, 0)), (300, 70001, 2051, (0, 0), (0, 0))])
def test_every_row_has_a_log_sum(ctx, rows, vocab, d, pads, offsets, ignored, dtype):
    """With a target or without; a row without one has a loss of 0. The losses are the same where lse is not asked for."""
    h, w, t, _ = inputs(rows, vocab, d, dtype, rows + vocab, ignored, pads=pads, offsets=offsets)
    (want_lse, err_lse), (want_loss, err_loss) = sums(h.t, w.t, t)
    loss, lse = forward(ctx, h, w, t)
    assert_within(lse, want_lse, err_lse, "lse")
    assert_within(loss, want_loss, err_loss, "loss")
    assert torch.equal(forward(ctx, h, w, t, ask=False)[0], loss)


def test_a_log_sum_for_bad_targets_and_in_a_graph(ctx):
    h, w, t, _ = inputs(200, 700, 72, torch.bfloat16, 3, 0.3)
    loss, lse = forward(ctx, h, w, t)
    again = forward(ctx, h, w, t, call=lambda f: replayed(ctx, f))
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)
    at = int(torch.nonzero(t < 0)[0])
    t[at] = 700
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        forward(ctx, h, w, t)


def test_what_rows_without_a_target_hold(ctx):
    """Their own log-sum alone depends on it; without lse they are not read, and the gradients never read them."""
    h, w, t, dloss = inputs(300, 500, 64, torch.bfloat16, 7, 0.4)
    site, none = fb.loss_site(300, 500, 64, torch.bfloat16), t == -1
    out = []
    for bad in (0.0, float("nan"), float("inf")):
        h.t[none] = bad
        (loss, lse), alone = forward(ctx, h, w, t), forward(ctx, h, w, t, ask=False)[0]
        assert torch.equal(loss, alone) and not loss[none].any()
        work = torch.full((ctx.linear_loss_workspace(site),), 0xFF, dtype=torch.uint8, device="cuda")
        dh, dw = torch.empty(300, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(500, 64, dtype=torch.bfloat16, device="cuda")
        ctx.linear_loss_grad(site, h.t, w.t, t, lse, torch.where(none, bad, dloss), dh, dw, work)
        assert torch.isfinite(lse[none]).any() == (bad == 0.0) and not dh[none].any()
        out.append((loss, lse[~none], dh, dw))
    for o in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], o))
    assert all(torch.isfinite(x).all() for x in out[0])


def test_scratch_off_16_bytes_is_refused(ctx):
    h, w, t, dloss = inputs(40, 300, 64, torch.bfloat16, 1)
    site = fb.loss_site(40, 300, 64, torch.bfloat16)
    buf, loss = torch.empty(ctx.linear_loss_workspace(site) + 64, dtype=torch.uint8, device="cuda"), torch.empty(40, device="cuda")
    for at in (1, 4, 8, 24):
        with pytest.raises(fb.MapalInfraError, match="16-byte boundary"):
            ctx.linear_loss(site, h.t, w.t, t, loss, loss, buf[at:])
        with pytest.raises(fb.MapalInfraError, match="16-byte boundary"):
            ctx.linear_loss_grad(site, h.t, w.t, t, loss, None, h.t, None, buf[at:])


@pytest.mark.parametrize("ask", [True, False])
@pytest.mark.parametrize("rows,vocab,spoilt", [(5, 129, slice(128, 129)), (40, 4000, slice(128, 256)), (3, 2, slice(1, 2)), (3, 2, slice(0, 1)),
                                               (40, 4000, slice(3999, 4000)), (40, 4000, slice(0, 4000)), (300, 9000, slice(0, 128)),
                                               (300, 9000, slice(7000, 7001)), (40, 300, slice(17, 18)), (40, 600, slice(256, 512))])
def test_a_logit_that_is_no_number_is_not_lost(ctx, rows, vocab, spoilt, ask):
    """Weights of NaN, the target's or others, in part of a tile of the vocabulary or in whole ones: every row's loss
    and lse are NaN, as the formula's. A row of h with a NaN spoils itself alone."""
    h, w, t, _ = inputs(rows, vocab, 72, torch.bfloat16, 2, 0.2 if rows > 5 else 0.0)
    clean = [x.clone() for x in forward(ctx, h, w, t, ask)]
    h.t[rows // 2, 5] = float("nan")
    loss, lse = forward(ctx, h, w, t, ask)
    there, other = t >= 0, torch.arange(rows, device="cuda") != rows // 2
    for got, was in zip((loss, lse), clean):
        assert torch.equal(got[other], was[other])
    assert torch.isnan(loss[rows // 2]) == there[rows // 2] and (not ask or torch.isnan(lse[rows // 2]))
    w.t[spoilt] = float("nan")
    loss, lse = forward(ctx, h, w, t, ask)
    assert torch.isnan(loss[there]).all() and not loss[~there].any() and (not ask or torch.isnan(lse).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("vocab", [2, 100, 129, 700, 5000])
def test_infinite_logits(ctx, vocab, dtype):
    """Weights of infinities and none of h at zero: lse is the limit, inf where a logit is, -inf where all are; the loss
    is inf where others outweigh the target, NaN where lse and the target's logit are the same infinity."""
    rows, d, inf = 12, 8, float("inf")
    h, w, t, _ = inputs(rows, vocab, d, dtype, 5)
    h.t.fill_(0)
    h.t[:, 0], h.t[::2, 1] = 1, 0.5
    h.t[:, 1] += 0.25
    t[:] = torch.arange(rows, device="cuda") % vocab
    t[rows - 1] = -1

    def holds(lse_want):
        loss, lse = forward(ctx, h, w, t)
        l = h.t.double() @ w.t.double().t()
        want = torch.logsumexp(l, 1)
        there = t >= 0
        want_loss = torch.where(there, want - l.gather(1, t.long().clamp(min=0)[:, None])[:, 0], 0.0)
        assert torch.isinf(want).all() == lse_want and not torch.isnan(want).any()
        assert_within(lse, want, torch.where(torch.isinf(want), 0.0, 1e-4), "lse")
        assert_within(loss, want_loss, torch.where(torch.isinf(want_loss), 0.0, 1e-4), "loss")

    w.t[:, 1] = 1
    w.t[vocab - 1, 0] = -inf  # a logit that adds nothing; a loss of inf for its own rows
    holds(False)
    w.t[1:, 0] = -inf
    holds(False)
    w.t[:, 0] = -inf
    holds(True)
    w.t[vocab - 1, 0] = inf
    holds(True)
    w.t[:, 0] = inf
    holds(True)


def exact_sums(h, w, t):
    """As sums(), for logits that are exact in f32: the exponent is off by two roundings of l*log2(e), the sum of
    exponentials by 2^-22 + 2^-19, lse and the loss by their own rounding."""
    (lse, _), (loss, _) = sums(h, w, t)
    big = (h.double() @ w.double().t()).abs().amax(1)
    err = 2 * 1.4427 * U32 * big + 2.0 ** -22 + 2.0 ** -19
    return (lse, err + U32 * lse.abs()), (loss, torch.where(t >= 0, err + 2 * U32 * (lse.abs() + loss.abs()), 0.0))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [1024, 2048, 2056, 4096])
@pytest.mark.parametrize("form", ["identical", "one channel", "powers of two"])
def test_logits_that_are_exact(ctx, form, d, dtype):
    """No sum of these rounds, however long: the vocabulary's rows are all the same (lse is l + log(vocab)), h has one
    channel each, or every product is the same power of two."""
    rows, vocab = 70, 700
    h, w, t, _ = inputs(rows, vocab, d, dtype, 4)
    r, v = torch.arange(rows, device="cuda"), torch.arange(vocab, device="cuda")
    if form == "identical":
        w.t[:] = 1 / 64
        h.t[:] = ((r % 5 - 2) / 2)[:, None]  # up to 64 at d = 4096
    elif form == "one channel":
        h.t.zero_()
        h.t[r, r * 37 % d] = 1
        w.t[:] = (torch.randint(-2048, 2048, (vocab, d), device="cuda") / 64).to(dtype)
    else:
        w.t[:] = (2.0 ** -(v % 3 + 6))[:, None]
        h.t[:] = (2.0 ** (r % 3 - 1))[:, None]
    (want_lse, err_lse), (want_loss, err_loss) = exact_sums(h.t, w.t, t)
    loss, lse = forward(ctx, h, w, t)
    assert_within(lse, want_lse, err_lse, "lse")
    assert_within(loss, want_loss, err_loss, "loss")


@pytest.mark.parametrize("where", ["first", "last", "spread"])
def test_a_sum_is_not_cut_whatever_its_order(ctx, where):
    """Logits of some 25 that a few channels make, first, last or among the others. In one sum on the tensor cores each
    of the d/16 steps cuts 2^-26 of what is there, in the mean: d/16 * 2^-26 of the logit where the large channels
    come first. At most a quarter of that is left in the mean of lse, as for sums of like channels."""
    rows, vocab, d, large = 256, 6000, 4096, 32
    g = torch.Generator(device="cuda").manual_seed(17)
    at = {"first": slice(0, large), "last": slice(d - large, d), "spread": slice(5, d, d // large)}[where]
    w = torch.randn(vocab, d, generator=g, device="cuda") / d ** 0.5
    h = torch.randn(rows, d, generator=g, device="cuda")
    w[:, at] = 0.75 + 0.1 * torch.rand(vocab, large, generator=g, device="cuda")
    h[:, at] = 1 + 0.1 * torch.rand(rows, large, generator=g, device="cuda")
    w, h = w.to(torch.bfloat16), h.to(torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    site = fb.loss_site(rows, vocab, d, torch.bfloat16)
    work = torch.empty(ctx.linear_loss_workspace(site, grad=False), dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(rows, device="cuda") for _ in range(2))
    ctx.linear_loss(site, h, w, t, loss, lse, work)
    l = h.double() @ w.double().t()
    want = torch.logsumexp(l, 1)
    average = (torch.softmax(l, 1) * l).sum(1).mean()
    assert average > 20 and (lse.double() - want).mean().abs() <= 0.25 * d / 16 * 2.0 ** -26 * average


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,offset", [(136, 0), (2048, 0), (4096, 0), (4099, 1)])
@pytest.mark.parametrize("order", [1, -1])
def test_the_gradient_of_nearly_certain_targets(ctx, order, d, offset, dtype):
    """1 - p of a target with a logit of some 20 that its first (or last) channels make, from the loss's own lse. Row i
    alone has channel i, of which the weights are 0, so that dw[:, i] is dl of row i, rounded twice (f16: at a scale
    that brings 1 to 2^14). lse is rounded by U32 of itself and the difference to it is exact; the others' sum has
    their logits' errors."""
    rows, vocab, large = 24, 5000, 48
    g = torch.Generator(device="cuda").manual_seed(23)
    h, w, t, _ = inputs(rows, vocab, d, dtype, 9, offsets=(0, offset))
    t[:] = torch.randperm(vocab, generator=g, device="cuda")[:rows]
    h.t.mul_(0.5)
    w.t.mul_(0.5)
    lead = torch.arange(rows, rows + large, device="cuda") if order > 0 else torch.arange(d - large, d, device="cuda")
    signs = torch.randint(0, 2, (rows, large), generator=g, device="cuda") * 2.0 - 1
    h.t[:, lead] = (signs * (0.6 + 0.1 * torch.rand(rows, large, generator=g, device="cuda"))).to(dtype)
    w.t[:, lead] = (0.1 * torch.randn(vocab, large, generator=g, device="cuda")).to(dtype)
    w.t[t.long()[:, None], lead] = (signs * 0.65).to(dtype)
    h.t[:, :rows] = torch.eye(rows, device="cuda").to(dtype)
    w.t[:, :rows] = 0
    site = fb.loss_site(rows, vocab, d, dtype, ldh=h.ld, ldw=w.ld)
    work = torch.empty(ctx.linear_loss_workspace(site, w=w.t), dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(rows, device="cuda") for _ in range(2))
    dh, dw = torch.empty(rows, d, dtype=dtype, device="cuda"), torch.empty(vocab, d, dtype=dtype, device="cuda")
    ctx.linear_loss(site, h.t, w.t, t, loss, lse, work)
    ctx.linear_loss_grad(site, h.t, w.t, t, lse, None, dh, dw, work)
    h64, w64, at = h.t.double(), w.t.double(), t.long()[:, None]
    l = h64 @ w64.t()
    p = torch.softmax(l, 1)
    missing = p.scatter(1, at, 0.0).sum(1)  # 1 - p of the target, without the difference
    assert missing.max() < 2e-3 and missing.min() < 2e-5
    size = (h64.abs() @ w64.abs().t()).amax(1)
    rel = (d + 16) * 17 / 16 * 2 * U32 * size + 8 * U32 * l.abs().amax(1) + 2.0 ** -18
    tiny = 2.0 ** -38 if dtype == torch.float16 else 0.0
    err = 2 * U32 * lse.double() + missing * (rel + 2 * half_step(dtype)) + tiny + out_error(missing, dtype)
    got = -dw[t.long(), torch.arange(rows, device="cuda")].double()
    assert_within(got, missing, err, "1 - p")
    others = p.scatter(1, at, 0.0).t()
    err = others * (2 * rel[None] + 2 * half_step(dtype)) + tiny + out_error(others, dtype)
    assert_within(dw[:, :rows].double().scatter(0, at.t(), 0.0), others, err, "p")

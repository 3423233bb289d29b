"""Products in 16-bit floats by expert and their gradients on a B200.

Most inputs here are small whole numbers: their products and sums up to 2^24 are
exact in f32 in any order, so outputs are compared bit for bit with the f64
formula rounded once. Random inputs are held to the sums' error bound."""
import pytest
import torch

import flow_b200 as fb
from _rows import U32, Guarded, assert_within, out_error, replayed

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def whole(shape, dtype, seed, most=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def ragged(m, groups, seed, behind=0):
    """Offsets of m - behind rows over groups, some of them empty."""
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, m - behind + 1, (groups - 1,), generator=g).sort().values
    if groups > 3:
        cuts[1] = cuts[0]
    return torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([m - behind])]).to(torch.int32).cuda()


def wants(x, w, dy, off):
    """y, dx, dw in f64; rows in no group are NaN."""
    x, w, dy = x.double(), w.double(), dy.double()
    y = torch.full((x.shape[0], w.shape[1]), float("nan"), dtype=torch.float64, device="cuda")
    dx = torch.full(x.shape, float("nan"), dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    ends = off.tolist() if off is not None else [0, x.shape[0]]
    for g in range(w.shape[0]):
        r = slice(ends[g], ends[g + 1])
        y[r], dx[r], dw[g] = x[r] @ w[g].t(), dy[r] @ w[g], dy[r].t() @ x[r]
    return y, dx, dw


def operands(m, n, k, groups, dtype, pads=(0, 0, 0), offsets=(0, 0, 0), seed=1):
    x = Guarded(m, k, dtype, pads[0], offsets[0]).put(whole((m, k), dtype, seed))
    w = Guarded(groups * n, k, dtype, pads[1], offsets[1]).put(whole((groups * n, k), dtype, seed + 1))
    dy = Guarded(m, n, dtype, pads[2], offsets[2]).put(whole((m, n), dtype, seed + 2))
    return x, w, dy


def check(ctx, m, n, k, groups, dtype, pads=(0, 0, 0), offsets=(0, 0, 0), behind=0, ytype=None, dwtype=None, seed=1,
          opads=(0, 0, 0), call=lambda f: f()):
    """All three products on whole numbers, bit for bit; what lies around the outputs stays as it was."""
    ytype, dwtype = ytype or dtype, dwtype or dtype
    x, w, dy = operands(m, n, k, groups, dtype, pads, offsets, seed)
    off = ragged(m, groups, seed + 3, behind) if groups > 1 or behind else None
    y, dx = Guarded(m, n, ytype, opads[0], opads[0]), Guarded(m, k, dtype, opads[1], opads[1])
    dw = Guarded(groups * n, k, dwtype, opads[2], opads[2])
    site = fb.product_site(m, n, k, dtype, groups=groups, ldx=x.ld, ldw=w.ld, ldy=y.ld, lddy=dy.ld, lddx=dx.ld,
                           lddw=dw.ld, ytype=ytype, dwtype=dwtype)
    for b in (y, dx, dw):
        b.t.fill_(77)

    def go():
        ctx.product(site, x.t, w.t, y.t, offsets=off)
        ctx.product_grad(site, x.t, w.t, dy.t, dx.t, dw.t, offsets=off)

    call(go)
    wy, wdx, wdw = wants(x.t, w.t.reshape(groups, n, k), dy.t, off)
    for got, want, what in ((y, wy, "y"), (dx, wdx, "dx"), (dw, wdw.reshape(groups * n, k), "dw")):
        exact = torch.where(torch.isnan(want), 77.0, want).to(torch.float32)  # whole numbers below 2^24
        assert exact.abs().max() < 2 ** 24 if exact.numel() else True
        want = exact.to(got.t.dtype)
        assert torch.equal(got.t, want), (what, (got.t.double() - want.double()).abs().max(),
                                          torch.nonzero(got.t != want)[:4].tolist())
        assert got.intact(), what


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 8, 8), (2, 3, 5), (4, 64, 64), (7, 100, 33), (16, 128, 256), (17, 129, 65),
                                   (100, 64, 1000), (128, 256, 64), (130, 300, 200), (255, 257, 259), (256, 256, 256),
                                   (513, 264, 520), (1000, 512, 136), (33, 2056, 72)])
def test_one_matrix(ctx, m, n, k, dtype):
    check(ctx, m, n, k, 1, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k,groups,behind", [
    (5, 16, 24, 2, 0), (40, 64, 64, 7, 3), (300, 136, 200, 5, 0), (1000, 128, 64, 64, 17), (777, 256, 512, 3, 100),
    (64, 33, 47, 40, 0), (2500, 264, 328, 9, 1), (3, 40, 40, 100, 1), (1, 64, 128, 5, 0), (513, 520, 72, 12, 513)])
def test_groups(ctx, m, n, k, groups, behind, dtype):
    check(ctx, m, n, k, groups, dtype, behind=behind)


@pytest.mark.parametrize("pads,offsets,opads", [((8, 8, 8), (0, 0, 0), (0, 0, 0)), ((1, 0, 0), (0, 0, 0), (1, 2, 3)),
                                                ((0, 3, 0), (0, 0, 0), (0, 0, 0)), ((0, 0, 5), (0, 0, 0), (8, 8, 8)),
                                                ((8, 16, 8), (1, 0, 0), (0, 0, 0)), ((8, 8, 8), (0, 7, 3), (3, 1, 2)),
                                                ((16, 8, 24), (8, 16, 24), (2, 0, 4))])
@pytest.mark.parametrize("m,n,k,groups", [(70, 64, 72, 1), (200, 136, 120, 3), (301, 257, 131, 4)])
def test_strides_and_places(ctx, m, n, k, groups, pads, offsets, opads):
    check(ctx, m, n, k, groups, torch.bfloat16, pads, offsets, opads=opads)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k,groups", [(40, 72, 64, 1), (600, 256, 320, 4), (33, 65, 31, 2)])
def test_f32_outputs(ctx, m, n, k, groups, dtype):
    check(ctx, m, n, k, groups, dtype, ytype=torch.float32, dwtype=torch.float32)


@pytest.mark.parametrize("m,n,k,groups", [(0, 8, 16, 3), (5, 0, 8, 2), (5, 8, 0, 2), (0, 0, 0, 1)])
def test_nothing(ctx, m, n, k, groups):
    """Empty arrays: sums over nothing are zeros."""
    t = torch.bfloat16
    off = torch.tensor([0] + [m] * groups, dtype=torch.int32, device="cuda")
    z = lambda *s: torch.full(s, 5.0, dtype=t, device="cuda")  # noqa: E731
    y, dx, dw = z(m, n), z(m, k), z(groups, n, k)
    site = fb.product_site(m, n, k, t, groups=groups)
    ctx.product(site, z(m, k), z(groups, n, k), y, offsets=off)
    ctx.product_grad(site, z(m, k), z(groups, n, k), z(m, n), dx, dw, offsets=off)
    for o in (y, dx, dw):
        assert not o.any()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k,groups", [(50, 200, 300, 1), (500, 256, 1024, 3), (301, 129, 513, 4), (2000, 512, 512, 2)])
def test_random(ctx, m, n, k, groups, dtype):
    """Products are exact in f32. Every one of a sum's depth/16 steps on the tensor cores adds 16 products to the sum
    so far, each of the 17 cut at one unit in the last place of a partial sum at most: 17/16*depth*2*U32 of the sum of
    absolute products; then one rounding."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, dy, off = r(m, k), r(groups, n, k), r(m, n), ragged(m, groups, 5) if groups > 1 else None
    for wide in (None, torch.float32):
        y = torch.empty(m, n, dtype=wide or dtype, device="cuda")
        dx, dw = torch.empty(m, k, dtype=dtype, device="cuda"), torch.empty(groups, n, k, dtype=wide or dtype, device="cuda")
        site = fb.product_site(m, n, k, dtype, groups=groups, ytype=wide, dwtype=wide)
        ctx.product(site, x, w, y, offsets=off)
        ctx.product_grad(site, x, w, dy, dx, dw, offsets=off)
        most = wants(x.abs(), w.abs(), dy.abs(), off)
        for got, want, top, depth in zip((y, dx, dw), wants(x, w, dy, off), most, (k, n, m)):
            err = (depth + 16) * 17 / 16 * 2 * U32 * top
            assert_within(got, want, err + out_error(want.abs() + err, got.dtype))


def test_not_numbers_stay_in_their_rows(ctx):
    """A row of NaN or infinities spoils its own row of y and dx and its group's dw, no others."""
    m, n, k, groups = 200, 64, 128, 4
    t = torch.bfloat16
    x, w, dy = whole((m, k), t, 1), whole((groups, n, k), t, 2), whole((m, n), t, 3)
    off = torch.tensor([0, 37, 90, 150, 190], dtype=torch.int32, device="cuda")
    x[90:] = float("nan")
    dy[195:] = float("inf")
    dy[90:190] = float("nan")
    y, dx, dw = torch.zeros(m, n, dtype=t, device="cuda"), torch.zeros(m, k, dtype=t, device="cuda"), torch.zeros(groups, n, k, dtype=t, device="cuda")
    site = fb.product_site(m, n, k, t, groups=groups)
    ctx.product(site, x, w, y, offsets=off)
    ctx.product_grad(site, x, w, dy, dx, dw, offsets=off)
    wy, wdx, wdw = wants(x[:90], w[:2], dy[:90], off[:3])
    assert torch.equal(y[:90].double(), wy.to(t).double()) and torch.equal(dx[:90].double(), wdx.to(t).double())
    assert torch.equal(dw[:2].double(), wdw.to(t).double())
    assert torch.isnan(y[90:190]).all() and torch.isnan(dx[90:190]).all() and torch.isnan(dw[2:]).all()
    assert not y[190:].any() and not dx[190:].any()  # in no group


@pytest.mark.parametrize("bad", [[0, 9, 5, 20], [0, 5, 9, 21], [-3, 5, 9, 20], [30, 40, 50, 60], [0, -7, 3, 20]])
def test_bad_offsets_trap(ctx, bad):
    m, n, k, t = 20, 64, 64, torch.float16
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    x, w, dy = operands(m, n, k, 3, t)
    y, dx, dw = Guarded(m, n, t, 8), Guarded(m, k, t, 8), Guarded(3 * n, k, t, 8)
    site = fb.product_site(m, n, k, t, groups=3, ldy=y.ld, lddx=dx.ld, lddw=dw.ld)
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.product(site, x.t, w.t, y.t, offsets=off)
    for a, b in ((dx.t, None), (None, dw.t)):
        with pytest.raises(fb.MapalTrap, match="index_oob"):
            ctx.product_grad(site, x.t, w.t, dy.t, a, b, offsets=off)
    assert y.intact() and dx.intact() and dw.intact()
    ctx.synchronize()


def test_one_gradient_alone(ctx):
    m, n, k, t = 100, 72, 64, torch.bfloat16
    x, w, dy = whole((m, k), t, 1), whole((1, n, k), t, 2), whole((m, n), t, 3)
    site = fb.product_site(m, n, k, t)
    _, wdx, wdw = wants(x, w, dy, None)
    dx, dw = torch.zeros(m, k, dtype=t, device="cuda"), torch.zeros(n, k, dtype=t, device="cuda")
    ctx.product_grad(site, None, w, dy, dx, None)
    assert torch.equal(dx, wdx.to(t)) and not dw.any()
    dx.zero_()
    ctx.product_grad(site, x, None, dy, None, dw)
    assert torch.equal(dw, wdw[0].to(t)) and not dx.any()


def test_captured(ctx):
    check(ctx, 700, 264, 520, 6, torch.bfloat16, behind=9, call=lambda f: replayed(ctx, f))


def test_two_streams():
    """Two contexts on streams of their own at once."""
    ctxs, streams = [fb.Context((0,), sync=False) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    t, m, n, k = torch.float16, 900, 520, 264
    x, w, dy = whole((m, k), t, 1), whole((4, n, k), t, 2), whole((m, n), t, 3)
    off = ragged(m, 4, 3)
    site = fb.product_site(m, n, k, t, groups=4)
    outs = [[torch.zeros(m, n, dtype=t, device="cuda"), torch.zeros(m, k, dtype=t, device="cuda"),
             torch.zeros(4, n, k, dtype=t, device="cuda")] for _ in ctxs]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s, (y, dx, dw) in zip(ctxs, streams, outs):
            c.set_stream(s.cuda_stream)
            c.product(site, x, w, y, offsets=off)
            c.product_grad(site, x, w, dy, dx, dw, offsets=off)
    for c in ctxs:
        c.synchronize()
    for got, want in zip(outs[0], wants(x, w, dy, off)):
        assert torch.equal(got, want.to(t))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k,groups,gap", [(300, 64, 72, 3, 1), (300, 65, 131, 3, 1), (90, 33, 47, 5, 2), (700, 257, 129, 2, 3)])
def test_matrices_apart(ctx, m, n, k, groups, gap, dtype):
    """Rows between one matrix and the next, which are left as they were in dw."""
    x, dy, off = whole((m, k), dtype, 1), whole((m, n), dtype, 2), ragged(m, groups, 3)
    buf = torch.full((groups, n + gap, k), float("nan"), dtype=dtype, device="cuda")
    w = buf[:, :n].copy_(whole((groups, n, k), dtype, 4))
    out = torch.full((groups, n + gap, k), 77.0, dtype=dtype, device="cuda")
    y, dx = torch.empty(m, n, dtype=dtype, device="cuda"), torch.empty(m, k, dtype=dtype, device="cuda")
    site = fb.product_site(m, n, k, dtype, groups=groups, ldg=(n + gap) * k, lddg=(n + gap) * k)
    ctx.product(site, x, w, y, offsets=off)
    ctx.product_grad(site, x, w, dy, dx, out[:, :n], offsets=off)
    wy, wdx, wdw = wants(x, w, dy, off)
    assert torch.equal(y, wy.to(dtype)) and torch.equal(dx, wdx.to(dtype)) and torch.equal(out[:, :n], wdw.to(dtype))
    assert (out[:, n:] == 77).all()


@pytest.mark.parametrize("m,n,k,groups", [(4096, 128, 128, 1), (3000, 136, 264, 2), (5000, 64, 200, 1), (2049, 512, 128, 3), (1100, 250, 131, 1)])
def test_long_sums_of_few_outputs(ctx, m, n, k, groups):
    """The weights' gradient of many rows and few weights, whose rows are cut over several CTAs; ragged groups, so that
    some cuts are empty and last blocks hold the next group's rows."""
    check(ctx, m, n, k, groups, torch.bfloat16, behind=7 if groups > 1 else 0)
    check(ctx, m, n, k, groups, torch.float16, ytype=torch.float32, dwtype=torch.float32, seed=9)


def test_past_two_to_the_31(ctx):
    """Operands and outputs of more than 2^31 elements: the last rows and the last matrix."""
    t, m, k, n = torch.bfloat16, 70000, 32768, 8
    x = torch.zeros(m, k, dtype=t, device="cuda")
    w, dy = whole((1, n, k), t, 1), whole((m, n), t, 2)
    x[-3:] = whole((3, k), t, 3)
    site = fb.product_site(m, n, k, t)
    y, dw = torch.empty(m, n, dtype=t, device="cuda"), torch.empty(1, n, k, dtype=t, device="cuda")
    ctx.product(site, x, w, y)
    ctx.product_grad(site, x, w, dy, None, dw)
    want, _, wdw = wants(x[-3:], w, dy[-3:], None)
    assert torch.equal(y[-3:], want.to(t)) and not y[:-3].any() and torch.equal(dw, wdw.to(t))
    ctx.product_grad(site, x, w, dy, x, None)  # dx into the rows
    _, wdx, _ = wants(torch.zeros(3, k, device="cuda"), w, dy[-3:], None)
    assert torch.equal(x[-3:], wdx.to(t))

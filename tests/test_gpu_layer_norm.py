"""Layer norm and its gradient on a B200 against the formulas in f64.

Bounds. U is half a step of f32, relative (2^-24). A row's sum is taken by at
least 32 threads and joined by a tree, so it has at most N = d/32 + 16
roundings on any value's path, and its error is at most N*U*sum|terms|; a sum
over rows has at most one rounding a row. Each bound below adds the errors of
the formula's parts to first order and half a step of the output's type."""
import pytest
import torch

import flow_b200 as fb
from _rows import TYPES, U32, Guarded, assert_within, out_error, replayed

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def rows_of(rows, d, dtype, seed, shift=0.0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, d, generator=g, device="cuda") * scale + shift).to(dtype)


def formula(x, w, b):
    x = x.double()
    mu = x.mean(1, keepdim=True)
    c = x - mu
    var = (c * c).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + EPS)
    w = torch.ones(x.shape[1], device="cuda", dtype=torch.float64) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    n = x.shape[1] / 32 + 16
    mu_err = n * U32 * x.abs().mean(1, keepdim=True) + U32 * mu.abs()
    # the variance around a mean that is off by mu_err is off by mu_err^2, and its sum rounds n times
    r_rel = 0.5 * r * r * (mu_err ** 2 + (n + 2) * U32 * var) + 4 * U32
    y = c * r * w + b
    err = w.abs() * (r * (mu_err + U32 * c.abs()) + (c * r).abs() * (r_rel + 2 * U32)) + U32 * (y.abs() + b.abs())
    return y, mu[:, 0], r[:, 0], err, mu_err[:, 0], (r * r_rel)[:, 0]


def grad_formula(x, w, mean, rstd, dy):
    """The gradient for the given f32 mean and rstd, and bounds of an f32 evaluation."""
    x, dy, rs = x.double(), dy.double(), rstd.double()[:, None]
    w = torch.ones(x.shape[1], device="cuda", dtype=torch.float64) if w is None else w.double()
    h, g = (x - mean.double()[:, None]) * rs, dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rs * (g - c1 - h * c2)
    n = x.shape[1] / 32 + 16
    e1 = (n + 2) * U32 * g.abs().mean(1, keepdim=True)
    e2 = (n + 5) * U32 * (g * h).abs().mean(1, keepdim=True)
    err = rs * (e1 + h.abs() * e2 + 6 * U32 * (g.abs() + c1.abs() + (h * c2).abs()))
    m = x.shape[0] + 20
    return dx, (dy * h).sum(0), dy.sum(0), err, (m + 3) * U32 * (dy * h).abs().sum(0), m * U32 * dy.abs().sum(0)


def run(ctx, x, w, b, y, dy=None, dx=None, wtype=None, dw=True, db=True, ldx=0, ldy=0, lddy=0, lddx=0):
    rows, d = x.shape
    f = lambda n: torch.full((n,), float("nan"), device="cuda")  # noqa: E731
    mean, rstd = f(rows), f(rows)
    site = fb.norm_site(rows, d, x.dtype, wdtype=wtype or (w.dtype if w is not None else x.dtype), eps=EPS, ldx=ldx,
                        ldy=ldy, lddy=lddy, lddx=lddx)
    ctx.layer_norm(site, x, w, b, y, mean, rstd)
    if dy is None:
        return mean, rstd
    gw, gb = f(d) if dw else None, f(d) if db else None
    work = torch.full((ctx.layer_norm_grad_workspace(site),), 255, dtype=torch.uint8, device="cuda")
    ctx.layer_norm_grad(site, x, w, mean, rstd, dy, dx, gw, gb, work if dw or db else None)
    return mean, rstd, gw, gb


def check(ctx, rows, d, dtype, wtype, affine=True, pad=0, offset=0, shift=0.0, scale=1.0, seed=1):
    gx = Guarded(rows, d, dtype, pad, offset).put(rows_of(rows, d, dtype, seed, shift, scale))
    gdy = Guarded(rows, d, dtype, pad, offset).put(rows_of(rows, d, dtype, seed + 1))
    gy, gdx = Guarded(rows, d, dtype, pad, offset), Guarded(rows, d, dtype, pad, offset)
    w = (rows_of(1, d, torch.float32, seed + 2)[0] * 0.3 + 1).to(wtype) if affine else None
    b = rows_of(1, d, torch.float32, seed + 3)[0].to(wtype) if affine else None
    ld = d + pad
    mean, rstd, dw, db = run(ctx, gx.t, w, b, gy.t, gdy.t, gdx.t, wtype, ldx=ld, ldy=ld, lddy=ld, lddx=ld)
    y, mu, r, y_err, mu_err, r_err = formula(gx.t, w, b)
    assert_within(mean, mu, mu_err + U32 * mu.abs(), "mean")
    assert_within(rstd, r, r_err + U32 * r, "rstd")
    assert_within(gy.t, y, y_err + out_error(y, dtype) * 1.01, "y")
    dx, gw, gb, dx_err, gw_err, gb_err = grad_formula(gx.t, w, mean, rstd, gdy.t)
    assert_within(gdx.t, dx, dx_err + out_error(dx, dtype) * 1.01, "dx")
    assert_within(dw, gw, gw_err, "dw")
    assert_within(db, gb, gb_err, "db")
    for g in (gx, gdy, gy, gdx):
        assert g.intact()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 31), (2, 33), (7, 64), (33, 127), (4, 256), (300, 257), (19, 1000),
                                    (1, 1024), (9, 1021), (6, 2048), (700, 1536), (5, 4096), (3, 5000), (2, 8192),
                                    (2, 8200), (3, 16384), (2, 16391), (2, 32768), (2, 33000), (1, 70001)])
def test_sizes(ctx, rows, d, dtype):
    check(ctx, rows, d, dtype, dtype)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("rows,d", [(5, 96), (40, 1023), (3, 4096), (2, 40000)])
def test_f32_weights(ctx, rows, d, dtype):
    check(ctx, rows, d, dtype, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (2, 2), (3, 5), (24, 8), (7, 4)])
@pytest.mark.parametrize("d", [50, 1024, 4095])
def test_strides_and_alignments(ctx, dtype, pad, offset, d):
    check(ctx, 11, d, dtype, dtype, pad=pad, offset=offset)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [40, 3000])
def test_without_weights(ctx, dtype, d):
    check(ctx, 13, d, dtype, dtype, affine=False)


@pytest.mark.parametrize("shift,scale", [(100.0, 1.0), (-30.0, 0.01), (0.0, 1e-4), (0.0, 200.0)])
@pytest.mark.parametrize("d", [200, 2500, 40000])
def test_far_means_and_small_variances(ctx, shift, scale, d):
    check(ctx, 6, d, torch.float32, torch.float32, shift=shift, scale=scale)
    check(ctx, 6, d, torch.bfloat16, torch.float32, shift=shift, scale=scale)


@pytest.mark.parametrize("d", [8, 1000, 4096, 40000])
def test_constant_rows(ctx, d):
    """A row of one value: the mean of equal values may round, and is then multiplied by 1/sqrt(eps)."""
    x = torch.full((4, d), 3.0, device="cuda")
    x[1] = 0.1
    x[2] = 0.0
    x[3] = -1e-30
    y = torch.empty_like(x)
    mean, rstd = run(ctx, x, None, None, y)
    want, mu, r, err, mu_err, r_err = formula(x, None, None)
    assert_within(y, want, err, "y")
    assert_within(mean, mu, mu_err + U32 * mu.abs(), "mean")
    assert torch.equal(y[2], torch.zeros_like(y[2]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 1001, 4096, 40000])
def test_rows_with_nan_and_infinity_stay_apart(ctx, dtype, d):
    x = rows_of(6, d, dtype, 3)
    x[1, d // 2] = float("nan")
    x[3, 0] = float("inf")
    x[4, d - 1] = float("-inf")
    y = torch.empty_like(x)
    run(ctx, x, None, None, y)
    for r in (1, 3, 4):
        assert torch.isnan(y[r]).any()
    ok = [0, 2, 5]
    want, _, _, err, _, _ = formula(x[ok], None, None)
    assert_within(y[ok], want, err + out_error(want, dtype) * 1.01, "y")


@pytest.mark.parametrize("rows", [0, 1, 2, 147, 149, 600, 5000])
@pytest.mark.parametrize("d", [72, 1024])
def test_row_counts(ctx, rows, d):
    if rows:
        check(ctx, rows, d, torch.bfloat16, torch.bfloat16)
        return
    x = torch.empty(0, d, device="cuda")
    _, _, dw, db = run(ctx, x, None, None, x, x, x)
    assert not dw.any() and not db.any()  # sums over no rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d,pad", [(80000, 64, 0), (76003, 63, 1), (40001, 128, 0), (39000, 127, 0), (20000, 256, 8), (16500, 300, 0),
                                        (9001, 600, 0), (5003, 1021, 3), (4903, 1024, 0), (2500, 2050, 0), (1203, 4096, 0),
                                        (1001, 5000, 0), (603, 8192, 0), (450, 12000, 0), (303, 16384, 0), (310, 16003, 0)])
def test_many_rows(ctx, rows, d, pad, dtype):
    check(ctx, rows, d, dtype, dtype, pad=pad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("rows,d", [(90001, 57), (60007, 121), (60003, 122), (22001, 249), (9003, 505), (4507, 1025), (2205, 2043),
                                    (1207, 4089), (1203, 4093), (603, 8185), (303, 8187), (203, 12001), (151, 16377)])
def test_rows_at_odd_places(ctx, rows, d, pad, dtype):
    """Rows that begin and end inside an access of 16 bytes: strides of every kind, neither the rows beside them
    nor the gaps between them written."""
    check(ctx, rows, d, dtype, torch.float32 if pad % 2 else dtype, pad=pad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 15, 17, 149, 600])
@pytest.mark.parametrize("d,pad", [(1, 0), (9, 0), (60, 1), (121, 0), (1021, 2), (8187, 0)])
def test_gradient_of_a_few_rows_at_odd_places(ctx, rows, d, pad, dtype):
    check(ctx, rows, d, dtype, dtype, pad=pad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(40001, 61), (4507, 1027)])
def test_values_beside_a_row_do_not_reach_it(ctx, dtype, rows, d):
    """Every other row holds NaN and infinities, which share accesses with the rows beside them."""
    x, dy = rows_of(rows, d, dtype, 3), rows_of(rows, d, dtype, 4)
    x[1::2, :7], x[1::2, -7:] = float("nan"), float("inf")
    dy[1::2] = float("nan")
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd, _, _ = run(ctx, x, None, None, y, dy, dx)
    assert torch.isnan(y[1::2]).all() and torch.isnan(dx[1::2]).all()
    x, dy, mean, rstd = x[::2], dy[::2], mean[::2], rstd[::2]
    want, _, _, err, _, _ = formula(x, None, None)
    assert_within(y[::2], want, err + out_error(want, dtype) * 1.01, "y")
    want, _, _, err, _, _ = grad_formula(x, None, mean, rstd, dy)
    assert_within(dx[::2], want, err + out_error(want, dtype) * 1.01, "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("strides", [(1021, 1029, 1037, 1021), (1024, 1021, 1021, 1024), (1022, 1026, 1022, 1030), (1021, 1022, 1023, 1024)])
def test_arrays_of_different_strides(ctx, dtype, strides):
    """Equal in where their rows begin, and not."""
    rows, d = 5003, 1021
    bufs = [torch.full((rows, ld), 7.0, device="cuda").to(dtype) for ld in strides]
    x, y, dy, dx = (b[:, :d] for b in bufs)
    x.copy_(rows_of(rows, d, dtype, 1))
    dy.copy_(rows_of(rows, d, dtype, 2))
    mean, rstd, dw, db = run(ctx, x, None, None, y, dy, dx, ldx=strides[0], ldy=strides[1], lddy=strides[2], lddx=strides[3])
    want, _, _, err, _, _ = formula(x, None, None)
    assert_within(y, want, err + out_error(want, dtype) * 1.01, "y")
    want, gw, gb, err, gw_err, gb_err = grad_formula(x, None, mean, rstd, dy)
    assert_within(dx, want, err + out_error(want, dtype) * 1.01, "dx")
    assert_within(dw, gw, gw_err, "dw")
    assert_within(db, gb, gb_err, "db")
    for b in bufs:
        assert (b[:, d:] == 7).all()


@pytest.mark.parametrize("rows,d", [(80001, 64), (70001, 59), (1203, 4093), (5003, 1021), (5003, 1024), (1203, 4096), (603, 8192), (303, 16384)])
def test_many_rows_in_place(ctx, rows, d):
    x, dy = rows_of(rows, d, torch.bfloat16, 5), rows_of(rows, d, torch.bfloat16, 6)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd, dw, db = run(ctx, x, None, None, y, dy, dx)
    site = fb.norm_site(rows, d, x.dtype, eps=EPS)
    work = torch.empty(ctx.layer_norm_grad_workspace(site), dtype=torch.uint8, device="cuda")
    dw2, db2 = torch.empty_like(dw), torch.empty_like(db)
    ctx.layer_norm_grad(site, x, None, mean, rstd, dy, dy, dw2, db2, work)
    ctx.layer_norm(site, x, None, None, x)
    assert torch.equal(dy, dx) and torch.equal(dw, dw2) and torch.equal(db, db2) and torch.equal(x, y)


def test_in_place(ctx):
    for d in (40, 1023, 4096, 20001, 70000):
        x, dy = rows_of(9, d, torch.float32, 5), rows_of(9, d, torch.float32, 6)
        w = rows_of(1, d, torch.float32, 7)[0]
        y, dx = torch.empty_like(x), torch.empty_like(x)
        mean, rstd, dw, db = run(ctx, x, w, None, y, dy, dx)
        site = fb.norm_site(9, d, x.dtype, eps=EPS)
        work = torch.empty(ctx.layer_norm_grad_workspace(site), dtype=torch.uint8, device="cuda")
        dw2, db2 = torch.empty_like(dw), torch.empty_like(db)
        ctx.layer_norm_grad(site, x, w, mean, rstd, dy, dy, dw2, db2, work)
        assert torch.equal(dy, dx) and torch.equal(dw, dw2) and torch.equal(db, db2)
        x2, dy = x.clone(), rows_of(9, d, torch.float32, 6)
        ctx.layer_norm_grad(site, x2, w, mean, rstd, dy, x2, dw2, db2, work)
        assert torch.equal(x2, dx) and torch.equal(dw, dw2) and torch.equal(db, db2)
        ctx.layer_norm(site, x, w, None, x)
        assert torch.equal(x, y)


def test_either_weight_gradient_alone(ctx):
    for d in (60, 2048, 40000):
        x, dy = rows_of(50, d, torch.bfloat16, 8), rows_of(50, d, torch.bfloat16, 9)
        y, dx = torch.empty_like(x), torch.empty_like(x)
        _, _, dw, db = run(ctx, x, None, None, y, dy, dx)
        dx2 = torch.empty_like(dx)
        _, _, one, none = run(ctx, x, None, None, y, dy, dx2, db=False)
        assert none is None and torch.equal(one, dw) and torch.equal(dx2, dx)
        _, _, none, one = run(ctx, x, None, None, y, dy, dx2, dw=False)
        assert none is None and torch.equal(one, db)
        dx2.zero_()
        run(ctx, x, None, None, y, dy, dx2, dw=False, db=False)
        assert torch.equal(dx2, dx)


@pytest.mark.parametrize("d", [24, 515, 2048])
def test_gradient_against_differences(ctx, d):
    """L = sum(y*dy): its change along v, by central differences of the f64 formula, is <dx, v> (and
    likewise for w and b). A central difference at step s of this L is off by s^2/6 times the third
    derivative, with v of the row's own size below 100 times the terms of L; s = 1e-4 leaves 2e-7."""
    x, dy = rows_of(8, d, torch.float32, 11), rows_of(8, d, torch.float32, 12)
    w, b = rows_of(1, d, torch.float32, 13)[0], rows_of(1, d, torch.float32, 14)[0]
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd, dw, db = run(ctx, x, w, b, y, dy, dx)
    vx, vw = rows_of(8, d, torch.float32, 15).double(), rows_of(1, d, torch.float32, 16)[0].double()
    L = lambda x, w, b: (formula(x, w, b)[0] * dy.double()).sum()  # noqa: E731
    s, x, w, b = 1e-4, x.double(), w.double(), b.double()
    scale = float((formula(x, w, b)[0] * dy.double()).abs().sum())
    diff = (L(x + s * vx, w, b) - L(x - s * vx, w, b)) / (2 * s)
    assert abs(float(diff - (dx.double() * vx).sum())) <= 2e-6 * scale
    diff = (L(x, w + s * vw, b) - L(x, w - s * vw, b)) / (2 * s)
    assert abs(float(diff - (dw.double() * vw).sum())) <= 2e-6 * scale
    diff = (L(x, w, b + s * vw) - L(x, w, b - s * vw)) / (2 * s)
    assert abs(float(diff - (db.double() * vw).sum())) <= 2e-6 * scale + 1e-9


def test_same_bits_every_time_and_other_streams(ctx):
    x, dy = rows_of(1000, 1536, torch.bfloat16, 21), rows_of(1000, 1536, torch.bfloat16, 22)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    first = [t.clone() for t in (*run(ctx, x, None, None, y, dy, dx), y, dx)]
    side = torch.cuda.Stream()
    old = ctx.stream()
    for stream in (None, side):
        y.zero_(), dx.zero_()
        torch.cuda.synchronize()
        if stream is not None:
            ctx.set_stream(stream.cuda_stream)
        again = (*run(ctx, x, None, None, y, dy, dx), y, dx)
        ctx.set_stream(old)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_captured_and_two_contexts(ctx):
    """A graph and eager calls of another context, each with scratch of its own, at once."""
    d = 2048
    x, dy = rows_of(400, d, torch.bfloat16, 31), rows_of(400, d, torch.bfloat16, 32)
    site = fb.norm_site(400, d, x.dtype, eps=EPS)

    def buffers():
        f = lambda n: torch.zeros(n, device="cuda")  # noqa: E731
        return dict(y=torch.zeros_like(x), mean=f(400), rstd=f(400), dx=torch.zeros_like(x), dw=f(d), db=f(d),
                    work=torch.zeros(ctx.layer_norm_grad_workspace(site), dtype=torch.uint8, device="cuda"))

    def step(c, o):
        c.layer_norm(site, x, None, None, o["y"], o["mean"], o["rstd"])
        c.layer_norm_grad(site, x, None, o["mean"], o["rstd"], dy, o["dx"], o["dw"], o["db"], o["work"])

    want, got, other = buffers(), buffers(), buffers()
    step(ctx, want)
    g = replayed(ctx, lambda: step(ctx, got), times=1)
    side = torch.cuda.Stream()
    with fb.Context((0,), sync=False) as c2:
        c2.set_stream(side.cuda_stream)
        for _ in range(5):
            g.replay()
            step(c2, other)
        c2.synchronize()
    torch.cuda.synchronize()
    for k in want:
        if k != "work":
            assert torch.equal(want[k], got[k]) and torch.equal(want[k], other[k]), k


def test_offsets_past_32_bits(ctx):
    """Rows whose elements lie more than 2^32 bytes and 2^31 elements into the buffer."""
    ld, d = (1 << 30) + 8, 1000
    x = torch.zeros(2 * ld + d, dtype=torch.float16, device="cuda")
    x = torch.as_strided(x, (3, d), (ld, 1))
    x.copy_(rows_of(3, d, torch.float16, 41))
    y, dy, dx = torch.empty(3, d, dtype=x.dtype, device="cuda"), rows_of(3, d, x.dtype, 42), torch.empty(3, d, dtype=x.dtype, device="cuda")
    mean, rstd, dw, db = run(ctx, x, None, None, y, dy, dx, ldx=ld)
    xc = x.contiguous()
    y2, dx2 = torch.empty_like(y), torch.empty_like(dx)
    run(ctx, xc, None, None, y2, dy, dx2)
    assert torch.equal(y, y2) and torch.equal(dx, dx2)


def test_short_workspace_is_refused(ctx):
    x = rows_of(64, 128, torch.float32, 1)
    site = fb.norm_site(64, 128, x.dtype)
    n = ctx.layer_norm_grad_workspace(site)
    f = torch.ones(128, device="cuda")
    with pytest.raises(fb.MapalInfraError, match="work is shorter"):
        ctx.layer_norm_grad(site, x, None, f, f, x, x.clone(), f.clone(), None,
                            torch.empty(n - 1, dtype=torch.uint8, device="cuda"))

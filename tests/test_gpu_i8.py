"""Rows to 8 bits and products in 8-bit integers on a B200.

The 8-bit values and the integer sums are exact, so nearly everything here is
compared bit for bit: torch evaluates the same f32 steps (one division, one
product, one rounding; a conversion and two products), and the sums are taken
in f64, which holds them."""
import pytest
import torch

import flow_b200 as fb
from _rows import TYPES, Guarded, replayed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def plain_quant(x):
    x = x.float()
    a = x.abs().amax(1, keepdim=True) if x.shape[1] else x.new_zeros(x.shape[0], 1)
    top = torch.full_like(a, 127.0)  # a tensor: torch divides by a number as a product with its reciprocal
    inv, scale = top / a, a / top
    tiny = torch.isinf(inv)
    inv, scale = torch.where(tiny, 0.0, inv), torch.where(tiny, 0.0, scale)
    odd = ~torch.isfinite(a)
    q = torch.where(tiny | odd, 0.0, torch.clamp(torch.round(x * inv), -127, 127))
    return q.to(torch.int8), torch.where(odd, float("nan"), scale)[:, 0]


def check_quant(ctx, x, pad=0, offset=0):
    rows, d = x.shape
    q = Guarded(rows, d, torch.int8, pad, offset)
    scale = torch.full((rows + 1,), 9.0, device="cuda")
    site = fb.quant_site(rows, d, x.dtype, ldx=x.stride(0) if rows > 1 else d, ldq=d + pad)
    ctx.quantize_rows_i8(site, x, q.t, scale)
    want, want_scale = plain_quant(x)
    assert torch.equal(q.t, want), (q.t.int() - want.int()).abs().max()
    assert torch.equal(torch.nan_to_num(scale[:rows], nan=-1.0), torch.nan_to_num(want_scale, nan=-1.0))
    assert scale[rows] == 9.0 and q.intact()


def rows_of(rows, d, dtype, seed=1, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, d, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (2, 3), (5, 16), (3, 100), (17, 512), (4, 1023), (600, 1024), (2000, 1028),
                                    (3, 4096), (9, 5001), (2, 8192), (3, 16384), (2, 20000), (2, 33333), (1, 70000)])
def test_quantize(ctx, dtype, rows, d):
    check_quant(ctx, rows_of(rows, d, dtype, rows + d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(90000, 64), (19000, 260), (9000, 1024), (5100, 1021), (5003, 1030), (2000, 4096), (1201, 5001),
                                    (700, 8192), (350, 16384), (320, 16001)])
def test_quantize_many_rows(ctx, dtype, rows, d):
    check_quant(ctx, rows_of(rows, d, dtype, rows + d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("xpad,pad", [(0, 0), (1, 1), (3, 0), (0, 7), (2, 6), (5, 13), (7, 8), (8, 4)])
@pytest.mark.parametrize("rows,d", [(40001, 57), (20003, 121), (9003, 1013), (4507, 1025), (2205, 2043), (1203, 4093), (603, 8185),
                                    (603, 8187), (301, 16369)])
def test_quantize_rows_at_odd_places(ctx, rows, d, xpad, pad, dtype):
    """Rows that begin and end inside an access; every third holds NaN and infinities, which share accesses with
    the rows beside it."""
    x = rows_of(rows, d, dtype, rows + d)
    x[1::3, :9], x[1::3, -9:] = float("nan"), float("inf")
    check_quant(ctx, Guarded(rows, d, dtype, xpad).put(x).t, pad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (4, 4), (16, 0), (7, 3), (8, 8)])
@pytest.mark.parametrize("d", [40, 1000, 4096])
def test_quantize_strides(ctx, dtype, pad, offset, d):
    x = Guarded(7, d, dtype, pad, offset).put(rows_of(7, d, dtype))
    check_quant(ctx, x.t, pad, offset)
    check_quant(ctx, x.t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 3001, 40000])
def test_quantize_odd_values(ctx, dtype, d):
    x = rows_of(12, d, dtype)
    x[1] = 0
    x[2, d - 1] = float("nan")
    x[3, 0] = float("inf")
    x[4, 5] = float("-inf")
    x[5] = -0.0
    x[6] = torch.finfo(dtype).max
    x[7] = -torch.finfo(dtype).smallest_normal
    x[8] = 0
    x[8, 3] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest subnormal
    x[9] = torch.arange(d, device="cuda").remainder(255).sub(127).mul(0.5)  # halves: ties go to the even
    x[10, 2], x[10, 3] = float("nan"), float("inf")
    if dtype is torch.float32:
        x[11] = 3.7e-37  # 127/a overflows just below 3.74e-37
        x[11, 1:] = 3.6e-37
    check_quant(ctx, x)


def test_quantize_nothing(ctx):
    scale = torch.full((3,), 9.0, device="cuda")
    e8, e = torch.empty(0, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda")
    ctx.quantize_rows_i8(fb.quant_site(0, 5, "float32"), e, e8, scale)
    assert (scale == 9).all()
    ctx.quantize_rows_i8(fb.quant_site(3, 0, "float32"), e, e8, scale)
    assert (scale == 0).all()


# ---- products ----------------------------------------------------------------------------------------------


def i8(shape, seed, lo=-128, hi=128):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device="cuda").to(torch.int8)


def f32(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def plain(A, sa, B, sb, dtype):
    acc = (A.double() @ B.double().t()).float()
    sa = torch.ones(A.shape[0], device="cuda") if sa is None else sa
    sb = torch.ones(B.shape[0], device="cuda") if sb is None else sb
    return (acc * sa[:, None] * sb[None, :]).to(dtype)


def check_mm(ctx, m, n, k, dtype, pads=(0, 0, 0), offsets=(0, 0, 0), A=None, B=None, seed=1):
    A = Guarded(m, k, torch.int8, pads[0], offsets[0]).put(i8((m, k), seed) if A is None else A)
    B = Guarded(n, k, torch.int8, pads[1], offsets[1]).put(i8((n, k), seed + 1) if B is None else B)
    C = Guarded(m, n, dtype, pads[2], offsets[2])
    sa, sb = f32(m, seed + 2) * 0.01, f32(n, seed + 3) * 0.01
    site = fb.matmul_i8_site(m, n, k, dtype, lda=k + pads[0], ldb=k + pads[1], ldc=n + pads[2])
    ctx.matmul_i8(site, A.t, sa, B.t, sb, C.t)
    want = plain(A.t, sa, B.t, sb, dtype)
    assert torch.equal(C.t, want), f"{int((C.t != want).sum())} cells differ"
    assert C.intact()


SHAPES = [(1, 1, 1), (1, 7, 16), (2, 3, 5), (1, 128, 128), (1, 4096, 512), (3, 200, 1000), (8, 129, 256), (16, 256, 2048),
          (17, 130, 100), (33, 64, 31), (64, 100, 64), (65, 300, 4096), (128, 128, 128), (128, 256, 129), (129, 257, 384),
          (200, 513, 1111), (256, 1000, 4096), (300, 96, 8192), (511, 640, 272), (1024, 1024, 1024), (700, 2300, 144)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ctx, dtype, m, n, k):
    check_mm(ctx, m, n, k, dtype)


# shapes that between them take every tile (channels x tokens) and splits of k over 1, 2, 4 and 8 blocks
CUTS = [(1, 32, 5520), (1, 4752, 32), (3, 2360, 8624), (97, 80, 5952), (944, 72, 48), (18, 2360, 10112), (117, 80, 6208),
        (2070, 72, 32), (603, 416, 9984), (623, 144, 6320), (168, 144, 6480), (66, 5176, 32), (1, 9528, 32),
        (1, 2392, 9824), (1, 1168, 6512), (17, 9808, 32), (21, 2424, 9024), (66, 456, 7008), (33, 9656, 32),
        (407, 664, 11024), (311, 456, 7712), (278, 200, 7328), (65, 13336, 32), (66, 8288, 32), (2500, 1000, 400),
        (5, 8192, 1024), (30, 4096, 896), (60, 8192, 384), (2100, 2056, 256)]


@pytest.mark.parametrize("m,n,k", CUTS)
def test_product_every_tile(ctx, m, n, k):
    check_mm(ctx, m, n, k, torch.bfloat16)
    check_mm(ctx, m, n, k, torch.float32, pads=(16, 32, 1))


@pytest.mark.parametrize("m,n,k", [(40, 300, 1009), (700, 260, 517), (2, 129, 4097), (1, 1, 300), (129, 1, 200), (1, 700, 77)])
@pytest.mark.parametrize("pads,offsets", [((0, 0, 0), (0, 0, 0)), ((1, 2, 0), (3, 7, 0)), ((5, 0, 0), (0, 9, 0)), ((16, 8, 0), (0, 0, 0))])
def test_product_unaligned(ctx, m, n, k, pads, offsets):
    check_mm(ctx, m, n, k, torch.bfloat16, pads, offsets)


def test_product_at_the_very_ends_of_its_buffers(ctx):
    """Unaligned operands that begin and end with their allocations (the loads of aligned words stay inside)."""
    for m, n, k in ((5, 130, 333), (150, 131, 1001)):
        A, B = i8((m, k), 1), i8((n, k), 2)
        C = torch.empty(m, n, device="cuda")
        ctx.matmul_i8(fb.matmul_i8_site(m, n, k, "float32"), A, None, B, None, C)
        assert torch.equal(C, plain(A, None, B, None, torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pads,offsets", [((16, 16, 0), (0, 0, 0)), ((16, 0, 8), (16, 16, 0)), ((0, 16, 1), (0, 32, 3)),
                                          ((1, 0, 0), (0, 0, 0)), ((0, 4, 0), (0, 0, 2)), ((8, 8, 2), (8, 8, 4)),
                                          ((0, 0, 0), (1, 0, 0)), ((0, 0, 0), (0, 4, 0)), ((3, 5, 7), (2, 6, 1))])
@pytest.mark.parametrize("m,n,k", [(4, 72, 160), (150, 200, 208), (300, 333, 128)])
def test_product_strides_and_alignments(ctx, dtype, pads, offsets, m, n, k):
    check_mm(ctx, m, n, k, dtype, pads, offsets)


@pytest.mark.parametrize("m,n,k", [(2, 40, 131071), (200, 140, 131056), (1, 3, 131070)])
def test_product_largest_sums(ctx, m, n, k):
    """Every product 128*128: the sum is 2^14*k, just below 2^31."""
    lowest = torch.full((max(m, n), k), -128, dtype=torch.int8, device="cuda")
    check_mm(ctx, m, n, k, torch.float32, A=lowest[:m], B=lowest[:n])
    high = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
    check_mm(ctx, m, n, k, torch.float32, A=lowest[:m], B=high)


def test_product_without_scales_and_nothing(ctx):
    A, B = i8((70, 96), 1), i8((130, 96), 2)
    C = torch.empty(70, 130, device="cuda")
    ctx.matmul_i8(fb.matmul_i8_site(70, 130, 96, "float32"), A, None, B, None, C)
    assert torch.equal(C, plain(A, None, B, None, torch.float32))
    for m in (1, 70):
        C.fill_(7)
        sa = f32(70, 3)
        sa[0] = float("inf")
        ctx.matmul_i8(fb.matmul_i8_site(m, 130, 0, "float32"), None, sa, None, None, C)
        assert torch.isnan(C[0]).all() and (C[1:m] == 0).all() and (C[m:] == 7).all()
    ctx.matmul_i8(fb.matmul_i8_site(0, 130, 96, "float32"), A, None, B, None, C)
    ctx.matmul_i8(fb.matmul_i8_site(70, 0, 96, "float32"), A, None, B, None, C)


def test_product_scales_that_are_not_finite(ctx):
    for m in (3, 200):
        A, B = i8((m, 64), 1, 1, 9), i8((150, 64), 2, 1, 9)
        sa, sb = f32(m, 3).abs() + 1, f32(150, 4).abs() + 1
        sa[1], sb[7] = float("nan"), float("inf")
        C = torch.empty(m, 150, dtype=torch.bfloat16, device="cuda")
        ctx.matmul_i8(fb.matmul_i8_site(m, 150, 64, "bfloat16"), A, sa, B, sb, C)
        want = plain(A, sa, B, sb, torch.bfloat16)
        assert torch.equal(torch.isnan(C), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(C), torch.nan_to_num(want))


def check_grouped(ctx, counts, n, k, dtype, tail=0, pads=(0, 0, 0), gap=0, first=0, seed=1):
    g, m = len(counts), first + sum(counts) + tail
    off = torch.tensor([first] + counts, device="cuda").cumsum(0).to(torch.int32)
    A = Guarded(m, k, torch.int8, pads[0]).put(i8((m, k), seed))
    ldb = k + pads[1]
    ldg = n * ldb + gap
    Bbuf = i8((g * ldg + 64,), seed + 1)
    B = torch.as_strided(Bbuf, (g, n, k), (ldg, ldb, 1))
    C = Guarded(m, n, dtype, pads[2], mark=5)
    sa, sb = f32(m, seed + 2) * 0.01, f32((g, n), seed + 3) * 0.01
    want = C.t.clone()
    lo = first
    for e, c in enumerate(counts):
        if c:
            want[lo:lo + c] = plain(A.t[lo:lo + c], sa[lo:lo + c], B[e], sb[e], dtype)
        lo += c
    site = fb.matmul_i8_site(m, n, k, dtype, groups=g, lda=k + pads[0], ldb=ldb, ldg=ldg, ldc=n + pads[2])
    ctx.matmul_i8(site, A.t, sa, B, sb, C.t, offsets=off)
    assert torch.equal(C.t, want), f"{int((C.t != want).sum())} cells differ"
    assert C.intact()


COUNTS = [[5], [0, 0, 3], [1] * 40, [0] * 7, [130, 1, 0, 200], [64, 128, 256, 1], [3, 0, 1, 2, 0, 0, 7, 1, 1, 0, 16, 2],
          [1000, 0, 0, 24], [127, 129, 128], [33] * 30, [0] * 50 + [300] + [0] * 50]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", COUNTS, ids=range(len(COUNTS)))
@pytest.mark.parametrize("n,k", [(128, 256), (200, 144), (77, 61)])
def test_grouped(ctx, dtype, counts, n, k):
    check_grouped(ctx, counts, n, k, dtype)


@pytest.mark.parametrize("counts", [[3, 0, 2], [140, 3, 0, 77]])
@pytest.mark.parametrize("pads,gap,first,tail", [((16, 16, 8), 0, 0, 9), ((0, 0, 0), 16, 0, 200), ((0, 16, 1), 160, 4, 3),
                                                 ((1, 0, 0), 0, 130, 1), ((0, 3, 0), 5, 2, 2), ((16, 16, 0), 8, 1, 1)])
def test_grouped_strides_and_rows_in_no_group(ctx, counts, pads, gap, first, tail):
    check_grouped(ctx, counts, 130, 272, torch.bfloat16, tail, pads, gap, first)


@pytest.mark.parametrize("g,m,n,k", [(2, 1, 32, 32), (60, 257, 40, 32), (60, 272, 72, 32), (60, 2514, 32, 32), (16, 2156, 136, 80),
                                     (60, 57, 136, 32), (60, 335, 136, 32), (60, 537, 136, 32), (16, 64, 1080, 32),
                                     (60, 1104, 136, 32), (3, 2000, 520, 256), (16, 3000, 264, 384)])
def test_grouped_every_tile(ctx, g, m, n, k):
    r = torch.Generator().manual_seed(m)
    counts = torch.bincount(torch.multinomial(torch.rand(g, generator=r), m, replacement=True, generator=r), minlength=g)
    check_grouped(ctx, counts.tolist(), n, k, torch.bfloat16)


def test_many_groups(ctx):
    counts = [(i * 7) % 4 for i in range(3000)]
    check_grouped(ctx, counts, 16, 32, torch.float32)


@pytest.mark.parametrize("off", [[0, 5, 3, 20], [0, 4, 8, 21], [-1, 4, 8, 20], [0, 1 << 30, 8, 20], [0, 4, 8, -9]])
@pytest.mark.parametrize("k", [64, 61])
def test_bad_offsets_trap_and_stay_inside(ctx, off, k):
    A, B, C = i8((20, k), 1), i8((3, 140, k), 2), Guarded(20, 140, torch.float32)
    off = torch.tensor(off, dtype=torch.int32, device="cuda")
    site = fb.matmul_i8_site(20, 140, k, "float32", groups=3)
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.matmul_i8(site, A, None, B, None, C.t, offsets=off)
    assert C.intact()
    off.copy_(torch.tensor([0, 5, 5, 20]))
    ctx.matmul_i8(site, A, None, B, None, C.t, offsets=off)  # the flag is clear again
    assert torch.equal(C.t[:5], plain(A[:5], None, B[0], None, torch.float32))


@pytest.mark.parametrize("off", [[0, 5, 3, 20], [0, 4, 8, 21], [-1, 4, 8, 20], [0, 1 << 30, 8, 20], [0, 9, -9, 12], [3, 2, 1, 15],
                                 [0, 3, 9] + [7] * 60 + [11, 10, 20]])
@pytest.mark.parametrize("k", [64, 61, 4096])
def test_bad_offsets_still_give_each_row_to_one_group(ctx, off, k):
    """An offset counts as the largest up to it, clamped; k = 4096 is split over a cluster."""
    g = len(off) - 1
    A, B, C = i8((20, k), 1), i8((g, 140, k), 2), torch.full((20, 140), 5.0, device="cuda")
    site = fb.matmul_i8_site(20, 140, k, "float32", groups=g)
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.matmul_i8(site, A, None, B, None, C, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
    want, top = torch.full_like(C, 5.0), [min(max(0, max(off[:i + 1])), 20) for i in range(len(off))]
    for e in range(g):
        if top[e + 1] > top[e]:
            want[top[e]:top[e + 1]] = plain(A[top[e]:top[e + 1]], None, B[e], None, torch.float32)
    assert torch.equal(C, want)


def test_offsets_that_go_up_and_down_cost_no_more_work(ctx):
    """Each of 4000 groups would otherwise claim all rows; the first takes them."""
    m, n, k, g = 2000, 256, 256, 4000
    A, B, C = i8((m, k), 1), i8((g, n, k), 2), torch.zeros(m, n, device="cuda")
    off = torch.tensor([0, m] * (g // 2) + [m], dtype=torch.int32, device="cuda")
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.matmul_i8(fb.matmul_i8_site(m, n, k, "float32", groups=g), A, None, B, None, C, offsets=off)
    assert torch.equal(C, plain(A, None, B[0], None, torch.float32))


@pytest.mark.parametrize("m", [3, 300])
def test_captured_replayed_and_two_contexts(ctx, m):
    A, B, sa, sb = i8((m, 512), 1), i8((2, 300, 512), 2), f32(m, 3), f32((2, 300), 4)
    C, C2 = (torch.zeros(m, 300, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    off = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    site = fb.matmul_i8_site(m, 300, 512, "bfloat16", groups=2)
    g = replayed(ctx, lambda: ctx.matmul_i8(site, A, sa, B, sb, C, offsets=off))
    off[1] = m // 3  # other routes and values in the same graph
    A.copy_(i8((m, 512), 9))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with fb.Context((0,), sync=False) as c2:
        c2.set_stream(side.cuda_stream)
        for _ in range(8):
            g.replay()
            c2.matmul_i8(site, A, sa, B, sb, C2, offsets=off)
        c2.synchronize()
    torch.cuda.synchronize()
    c = m // 3
    want = torch.cat([plain(A[:c], sa[:c], B[0], sb[0], torch.bfloat16), plain(A[c:], sa[c:], B[1], sb[1], torch.bfloat16)])
    assert torch.equal(C, want) and torch.equal(C2, want)


@pytest.mark.parametrize("m", [2, 3, 130])
def test_offsets_past_32_bits(ctx, m):
    """Rows of A more than 2^31 bytes apart, a second matrix of B past 2^31, rows of C past 2^32 bytes."""
    k, n = 160, 40
    lda = (1 << 31) // max(1, m - 1) // 16 * 16 + 16
    A = torch.as_strided(torch.zeros((m - 1) * lda + k, dtype=torch.int8, device="cuda"), (m, k), (lda, 1))
    A.copy_(i8((m, k), 1))
    ldg = (1 << 31) + 160
    B = torch.as_strided(torch.zeros(ldg + n * k, dtype=torch.int8, device="cuda"), (2, n, k), (ldg, k, 1))
    B.copy_(i8((2, n, k), 2))
    ldc = (1 << 30) // max(1, m - 1) // 8 * 8 + 8
    C = torch.as_strided(torch.zeros((m - 1) * ldc + n, device="cuda"), (m, n), (ldc, 1))
    off = torch.tensor([0, 1, m], dtype=torch.int32, device="cuda")
    ctx.matmul_i8(fb.matmul_i8_site(m, n, k, "float32", groups=2, lda=lda, ldg=ldg, ldc=ldc), A, None, B, None, C, offsets=off)
    assert torch.equal(C[:1], plain(A[:1], None, B[0], None, torch.float32))
    assert torch.equal(C[1:], plain(A[1:], None, B[1], None, torch.float32))

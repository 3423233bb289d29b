"""Dropout with a mask that is never stored, on a B200: the mask bit for bit against Philox 4x32-10 in numpy, values
within one rounding."""
import numpy as np
import pytest
import torch

import flow_b200 as fb
from _rows import TYPES, U32, Guarded, assert_within, out_error, replayed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def philox(c, k):
    """c: four uint32 arrays, k: two numbers (the method of Salmon et al., 2011)."""
    c, k = [x.astype(np.uint64) for x in c], [int(x) for x in k]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [x.astype(np.uint32) for x in c]


def bits(rng, rows, d):
    """The 16 bits of each element."""
    key, place = (int(v) % 2 ** 64 for v in rng.tolist())
    n = (d + 7) // 8
    col, row = np.meshgrid(np.arange(n, dtype=np.uint32), np.arange(rows, dtype=np.uint32))
    one = np.ones_like(col)
    w = philox([col, row, one * np.uint32(place & 0xFFFFFFFF), one * np.uint32(place >> 32)], (key & 0xFFFFFFFF, key >> 32))
    return np.stack([h for x in w for h in (x & 0xFFFF, x >> 16)], -1).reshape(rows, n * 8)[:, :d]


def test_known_answers(ctx):
    """The method's published answers: counter and key of zeros, and of ones. Thresholds cut the 16 bits out."""
    for ones, want in ((0, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),):
        halves = np.array([h for w in want for h in (w & 0xFFFF, w >> 16)])
        rng = torch.full((2,), ones, dtype=torch.int64, device="cuda")
        assert (bits(rng, 1, 8)[0] == halves).all()
        x, y = torch.ones(1, 8, device="cuda"), torch.empty(1, 8, device="cuda")
        for cut in sorted(set(halves.tolist()) | {int(h) + 1 for h in halves}):
            ctx.dropout(fb.dropout_site(1, 8, torch.float32, cut / 65536), x, None, y, rng)
            assert ((y[0] > 0).cpu().numpy() == (halves >= cut)).all()


def check(ctx, rows, d, dtype, p, pads=(0, 0, 0), offsets=(0, 0, 0), residual=True, seed=1, call=lambda f: f(), alias=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = Guarded(rows, d, dtype, pads[0], offsets[0]).put(torch.randn(rows, d, generator=g, device="cuda"))
    r = Guarded(rows, d, dtype, pads[1], offsets[1]).put(torch.randn(rows, d, generator=g, device="cuda")) if residual else None
    y = {None: lambda: Guarded(rows, d, dtype, pads[2], offsets[2]), "x": lambda: x, "residual": lambda: r}[alias]()
    rng = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), generator=g, device="cuda")
    limit = round(p * 65536)
    keep = torch.from_numpy(bits(rng, rows, d) >= limit).cuda()
    scale = float(np.float32(65536 / (65536 - limit))) if limit < 65536 else 0.0
    add = r.t.double() if residual else torch.zeros(rows, d, dtype=torch.float64, device="cuda")
    want = torch.where(keep, x.t.double() * scale, 0.0) + add
    ctx_site = fb.dropout_site(rows, d, dtype, p, ldx=x.ld, ldr=r.ld if residual else 0, ldy=y.ld)
    call(lambda: ctx.dropout(ctx_site, x.t, r.t if residual else None, y.t, rng))
    assert_within(y.t, want, out_error(want, dtype) * (1 + 2 * U32) + U32 * want.abs())
    assert x.intact() and y.intact()
    if not residual:
        assert torch.equal(y.t != 0, keep & (x.t != 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 7), (3, 8), (2, 9), (5, 64), (17, 100), (100, 1000), (33, 1021), (9, 4096), (3, 20001),
                                    (5000, 3), (2000, 264)])
def test_sizes(ctx, rows, d, residual, dtype):
    check(ctx, rows, d, dtype, 0.3, residual=residual, seed=rows + d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pads,offsets", [((8, 8, 8), (0, 0, 0)), ((1, 0, 2), (0, 0, 0)), ((0, 0, 0), (1, 2, 3)), ((4, 12, 8), (4, 8, 0)),
                                          ((2, 2, 2), (2, 2, 2)), ((7, 5, 3), (1, 6, 4))])
@pytest.mark.parametrize("rows,d", [(40, 136), (301, 1021), (7, 2050)])
def test_strides_and_places(ctx, rows, d, pads, offsets, dtype):
    check(ctx, rows, d, dtype, 0.25, pads, offsets)


@pytest.mark.parametrize("p", [0.0, 1e-6, 1 / 65536, 0.1, 0.5, 0.9, 65535 / 65536, 1.0])
def test_shares(ctx, p):
    check(ctx, 300, 500, torch.float32, p)


@pytest.mark.parametrize("alias", ["x", "residual"])
@pytest.mark.parametrize("rows,d", [(100, 256), (33, 1021)])
def test_in_place(ctx, alias, rows, d):
    check(ctx, rows, d, torch.bfloat16, 0.4, alias=alias)


def test_dropped_values_do_not_matter(ctx):
    """NaN and infinities where nothing is kept leave no trace."""
    rng = torch.tensor([5, 9], device="cuda")
    keep = torch.from_numpy(bits(rng, 64, 200) >= 32768).cuda()
    x = torch.where(keep, 1.0, float("nan"))
    x[::2] = torch.where(keep, 1.0, float("inf"))[::2]
    y = torch.empty(64, 200, device="cuda")
    ctx.dropout(fb.dropout_site(64, 200, torch.float32, 0.5), x, None, y, rng)
    assert torch.equal(y, torch.where(keep, 2.0, 0.0))


def test_the_gradient_has_the_same_mask(ctx):
    rng = torch.tensor([-3, 1 << 40], device="cuda")
    a, b = torch.ones(50, 333, device="cuda"), torch.ones(50, 340, dtype=torch.bfloat16, device="cuda")
    y, dx = torch.empty(50, 333, device="cuda"), torch.empty(50, 340, dtype=torch.bfloat16, device="cuda")
    ctx.dropout(fb.dropout_site(50, 333, torch.float32, 0.5), a, None, y, rng)
    ctx.dropout(fb.dropout_site(50, 333, torch.bfloat16, 0.5, ldx=340, ldy=340), b[:, :333], None, dx[:, :333], rng)
    assert torch.equal(y, dx[:, :333].float()) and 0.4 < (y > 0).float().mean() < 0.6


def test_captured_replays_follow_the_generator(ctx):
    x, y = torch.ones(64, 512, device="cuda"), torch.empty(64, 512, device="cuda")
    rng = torch.tensor([7, 0], device="cuda")
    site = fb.dropout_site(64, 512, torch.float32, 0.5)
    g = replayed(ctx, lambda: ctx.dropout(site, x, None, y, rng))
    for place in (0, 1, 2):
        rng[1] = place
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal((y > 0).cpu(), torch.from_numpy(bits(rng, 64, 512) >= 32768))


def test_past_two_to_the_31(ctx):
    """More than 2^31 elements."""
    rows, d = 70000, 32768
    x = torch.ones(rows, d, dtype=torch.bfloat16, device="cuda")
    rng = torch.tensor([11, 12], device="cuda")
    ctx.dropout(fb.dropout_site(rows, d, torch.bfloat16, 0.5), x, None, x, rng)
    at = [0, 1, 65535, 65537, rows - 1]
    b = bits(rng, rows, 64)[at] >= 32768
    assert torch.equal((x[at, :64] > 0).cpu(), torch.from_numpy(b))

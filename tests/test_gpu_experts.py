"""Rows sorted by expert and back, with weights and gradients, on a B200.

Places are whole numbers and compared exactly with a loop over the slots; moved
rows are compared bit for bit. A weighted sum of k terms in f32 has at most
k + 1 roundings of each term, a dot product of d terms d/32 + 16 (at least 32
threads a row and a tree), each of 2^-24 relative to the terms' sizes, and
outputs of 16 bits round once more."""
import numpy as np
import pytest
import torch

import flow_b200 as fb
from _rows import TYPES, U32, Guarded, assert_within, half_step, out_error, replayed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


def i32(n, fill=-7):
    return torch.full((n,), fill, dtype=torch.int32, device="cuda")


def plain_sort(ids, experts):
    ids = np.asarray(ids)
    there = np.nonzero((ids >= 0) & (ids < experts))[0]
    order = there[np.argsort(ids[there], kind="stable")]
    pos = np.full(ids.size, -1, np.int64)
    pos[order] = np.arange(order.size)
    return np.searchsorted(ids[order], np.arange(experts + 1)), order, pos


def sort(ctx, ids, experts, k=1):
    n = ids.numel()
    off, order, pos = i32(experts + 3), i32(n + 2), i32(n + 2)
    ctx.expert_sort(fb.expert_site(n // k, k, experts, 1, "float32"), ids, off, order, pos)
    return off, order, pos


def check_sort(ctx, ids, experts, k=1):
    off, order, pos = sort(ctx, ids, experts, k)
    w_off, w_order, w_pos = plain_sort(ids.cpu(), experts)
    n, m = ids.numel(), w_order.size
    assert np.array_equal(off.cpu()[:experts + 1], w_off) and (off[experts + 1:] == -7).all()
    assert np.array_equal(pos.cpu()[:n], w_pos) and (pos[n:] == -7).all()
    assert np.array_equal(order.cpu()[:m], w_order) and (order[m:] == -7).all()  # behind the last: left


def random_ids(n, experts, seed, drop=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, experts, (n,), generator=g, device="cuda", dtype=torch.int32)
    if drop:
        ids[torch.rand(n, generator=g, device="cuda") < drop] = -1
    return ids


@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 255, 1000, 4096, 4097, 8193, 16384, 16385, 50001, 262145, 1 << 20])
@pytest.mark.parametrize("experts", [1, 2, 8, 33, 256, 1000, 1024])
def test_sort(ctx, n, experts):
    check_sort(ctx, random_ids(n, experts, n + experts), experts)


@pytest.mark.parametrize("n", [7, 5000, 40000])
@pytest.mark.parametrize("drop", [0.1, 0.9, 1.0])
def test_sort_with_dropped_slots(ctx, n, drop):
    check_sort(ctx, random_ids(n, 60, n, drop), 60)


@pytest.mark.parametrize("n", [40, 5000, 70000])
def test_sort_one_expert_takes_all(ctx, n):
    check_sort(ctx, torch.full((n,), 63, dtype=torch.int32, device="cuda"), 64)
    check_sort(ctx, torch.zeros(n, dtype=torch.int32, device="cuda"), 64)
    check_sort(ctx, torch.arange(n, dtype=torch.int32, device="cuda") % 64, 64)


@pytest.mark.parametrize("bad", [64, 1 << 30, -2, -(1 << 31)])
def test_sort_traps_on_a_foreign_expert(ctx, bad):
    ids = random_ids(3000, 64, 5)
    ids[1717] = bad
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        sort(ctx, ids, 64)
    ids[1717] = 0  # the flag is clear again
    check_sort(ctx, ids, 64)


def test_sort_trap_of_a_replay_surfaces(ctx):
    ids = random_ids(500, 8, 5)
    off, order, pos = i32(9), i32(500), i32(500)
    site = fb.expert_site(500, 1, 8, 1, "float32")
    g = replayed(ctx, lambda: ctx.expert_sort(site, ids, off, order, pos))
    ctx.synchronize()
    ids[7] = 8
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(fb.MapalTrap):
        ctx.synchronize()
    ctx.synchronize()
    ids.copy_(random_ids(500, 8, 6))
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(pos.cpu(), plain_sort(ids.cpu(), 8)[2])


# ---- rows --------------------------------------------------------------------------------------------


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


class Layer:
    """Tokens, their places and the rows on both sides, all inside marked buffers."""

    def __init__(self, ctx, tokens, k, experts, d, dtype, drop=0.0, pad=0, offset=0, seed=1, spare=3):
        self.ctx, self.tokens, self.k, self.d, self.dtype = ctx, tokens, k, d, dtype
        n = tokens * k
        ids = random_ids(n, experts, seed, drop)
        off, _, self.pos = sort(ctx, ids, experts, k)
        self.pos = self.pos[:n]
        self.there = int(off[experts])
        self.w = randn((tokens, k), torch.float32, seed + 1)
        self.site = fb.expert_site(tokens, k, experts, d, dtype, rows=n + spare, ldt=d + pad, ldr=d + pad)
        self.T = lambda s=None: self._rows(tokens, pad, offset, s)  # noqa: E731
        self.R = lambda s=None: self._rows(n + spare, pad, offset, s)  # noqa: E731
        self.p = self.pos.long().view(tokens, k)
        self.in_ = (self.p >= 0)[..., None]

    def _rows(self, rows, pad, offset, seed):
        g = Guarded(rows, self.d, self.dtype, pad, offset, mark=5)
        return g if seed is None else g.put(randn((rows, self.d), self.dtype, seed))

    def picked(self, rows):
        """rows[pos] in f64, zeros where a slot has no place: tokens x k x d."""
        return torch.where(self.in_, rows.double()[self.p.clamp(min=0)], 0.0)


CASES = [(1, 1, 1, 1), (3, 2, 4, 5), (16, 8, 128, 256), (40, 3, 7, 1001), (5, 1, 9, 4096), (130, 4, 16, 515),
         (2, 17, 40, 64), (300, 2, 8, 1024), (7, 8, 8, 8200), (9, 40, 64, 96)]


@pytest.mark.parametrize("dtype", TYPES + [torch.int8])
@pytest.mark.parametrize("tokens,k,experts,d", CASES)
@pytest.mark.parametrize("pad,offset,drop", [(0, 0, 0.0), (1, 1, 0.3), (16, 0, 0.9)])
def test_dispatch(ctx, dtype, tokens, k, experts, d, pad, offset, drop):
    q = dtype is torch.int8
    L = Layer(ctx, tokens, k, experts, d, dtype, drop, pad, offset)
    x, xs = L.T(None if q else 3), L.R()
    if q:
        x.put(torch.randint(-128, 128, (tokens, d), device="cuda").to(torch.int8))
    scale, scale_out = randn(tokens, torch.float32, 4), torch.full((tokens * k + 3,), 9.0, device="cuda")
    want, want_scale = xs.t.clone(), scale_out.clone()
    for t in range(tokens):
        for j in range(k):
            if L.p[t, j] >= 0:
                want[L.p[t, j]], want_scale[L.p[t, j]] = x.t[t], scale[t]
    ctx.expert_dispatch(L.site, x.t, L.pos, xs.t, scale, scale_out)
    assert torch.equal(xs.t, want) and torch.equal(scale_out, want_scale)  # rows behind the last are left
    assert x.intact() and xs.intact()
    xs2 = L.R()
    ctx.expert_dispatch(L.site, x.t, L.pos, xs2.t)
    assert torch.equal(xs2.t, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,experts,d", CASES)
@pytest.mark.parametrize("pad,offset,drop", [(0, 0, 0.0), (1, 1, 0.3), (2, 2, 0.9), (8, 0, 0.2)])
def test_combine_and_gradients(ctx, dtype, tokens, k, experts, d, pad, offset, drop):
    L = Layer(ctx, tokens, k, experts, d, dtype, drop, pad, offset)
    h, y, dy, dh, dxs, dx = L.R(3), L.T(), L.T(4), L.R(), L.R(5), L.T()
    w = torch.where(L.in_[..., 0], L.w, float("nan"))  # the weight of a slot without a place is never used
    dw = torch.full((tokens, k), 9.0, device="cuda")
    before = dh.t.clone()
    ctx.expert_combine(L.site, h.t, w, L.pos, y.t)
    ctx.expert_combine_grad(L.site, h.t, w, L.pos, dy.t, dh.t, dw)
    ctx.expert_dispatch_grad(L.site, dxs.t, L.pos, dx.t)

    terms = L.w.double()[..., None] * L.picked(h.t)
    want = terms.sum(1)
    assert_within(y.t, want, (k + 1) * U32 * terms.abs().sum(1) + out_error(want, dtype) * 1.01, "y")
    terms = L.picked(dxs.t)
    want = terms.sum(1)
    assert_within(dx.t, want, (k + 1) * U32 * terms.abs().sum(1) + out_error(want, dtype) * 1.01, "dx")
    terms = dy.t.double()[:, None, :] * L.picked(h.t)
    assert_within(dw, terms.sum(2), (d / 32 + 16) * U32 * terms.abs().sum(2), "dw")
    assert (dw[~L.in_[..., 0]] == 0).all()
    got = L.picked(dh.t)
    want = torch.where(L.in_, L.w.double()[..., None] * dy.t.double()[:, None, :], 0.0)
    assert_within(got, want, U32 * want.abs() + out_error(want, dtype) * 1.01, "dh")
    assert torch.equal(dh.t[L.there:], before[L.there:])
    for g in (h, y, dy, dh, dxs, dx):
        assert g.intact()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,d", [(1500, 3, 200), (1300, 5, 1031), (1201, 4, 2048), (1190, 9, 72)])
def test_many_tokens(ctx, dtype, tokens, k, d):
    test_combine_and_gradients(ctx, dtype, tokens, k, 30, d, 0, 0, 0.1)


def test_more_rows_than_a_grid_has_blocks(ctx):
    n = (1 << 20) + 1111
    pos = torch.randperm(n, device="cuda").to(torch.int32)
    site = fb.expert_site(n, 1, 4, 3, "float32")
    x, w = randn((n, 3), torch.float32, 1), randn((n, 1), torch.float32, 2)
    xs, y, dh, dw = (torch.empty(n, 3, device="cuda") for _ in range(4))
    dw = torch.empty(n, 1, device="cuda")
    ctx.expert_dispatch(site, x, pos, xs)
    assert torch.equal(xs[pos.long()], x)
    ctx.expert_combine(site, xs, None, pos, y)
    assert torch.equal(y, x)
    ctx.expert_combine_grad(site, xs, w, pos, y, dh, dw)
    assert torch.equal(dh[pos.long()], w * x)
    assert_within(dw[:, 0], (x.double() ** 2).sum(1), 17 * U32 * (x.double() ** 2).sum(1), "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [50, 1400])
def test_without_weights_and_in_place(ctx, dtype, tokens):
    L = Layer(ctx, tokens, 3, 9, 136, dtype, 0.2)
    h, y, dx, dy = L.R(3), L.T(), L.T(), L.T(4)
    ctx.expert_combine(L.site, h.t, None, L.pos, y.t)
    ctx.expert_dispatch_grad(L.site, h.t, L.pos, dx.t)
    assert torch.equal(y.t, dx.t)
    dh, dw, dw2 = L.R(), torch.empty(tokens, 3, device="cuda"), torch.empty(tokens, 3, device="cuda")
    ctx.expert_combine_grad(L.site, h.t, None, L.pos, dy.t, dh.t, dw)
    ones = torch.ones(tokens, 3, device="cuda")
    dh2 = L.R()
    ctx.expert_combine_grad(L.site, h.t, ones, L.pos, dy.t, dh2.t, None)
    assert torch.equal(dh.t, dh2.t)
    ctx.expert_combine_grad(L.site, h.t, ones, L.pos, dy.t, h.t, dw2)  # dh is h
    assert torch.equal(dw, dw2) and torch.equal(h.t[:L.there], dh.t[:L.there])


def test_gradient_against_differences(ctx):
    """combine is linear in h and in w, so a difference over any step is its derivative: with
    L = sum(y*dy), L(h + v) - L(h) = <dh, v> and L(w + v) - L(w) = <dw, v>, up to rounding: y's own, a
    term's k + 2 and the products' of dh and dw, all relative to the terms' sizes."""
    L = Layer(ctx, 60, 4, 10, 300, torch.float32, 0.2)
    h, dy, y = L.R(3), L.T(4), L.T()
    dh, dw = L.R(), torch.empty(60, 4, device="cuda")
    ctx.expert_combine_grad(L.site, h.t, L.w, L.pos, dy.t, dh.t, dw)
    v, vw = randn(h.t.shape, torch.float32, 6), randn((60, 4), torch.float32, 7)
    vw[~L.in_[..., 0]] = 0

    def loss(hh, ww):
        ctx.expert_combine(L.site, hh, ww, L.pos, y.t)
        return float((y.t.double() * dy.t.double()).sum())

    # h + v and w + vw round once each, which is one more step relative to the terms
    size = float((L.w.abs().double()[..., None] * L.picked(h.t.abs() + v.abs()) * dy.t.abs().double()[:, None]).sum())
    diff = loss((h.t + v).contiguous(), L.w) - loss(h.t.contiguous(), L.w)
    assert abs(diff - float((L.picked(dh.t) * L.picked(v)).sum())) <= 2 * (4 + 4) * U32 * size
    size = float(((L.w.abs() + vw.abs()).double()[..., None] * L.picked(h.t).abs() * dy.t.abs().double()[:, None]).sum())
    diff = loss(h.t, L.w + vw) - loss(h.t, L.w)
    assert abs(diff - float((dw.double() * vw.double()).sum())) <= (2 * (4 + 4) + 300 / 32 + 16) * U32 * size


@pytest.mark.parametrize("bad", [53, 1 << 30])
def test_places_outside_trap_and_write_nothing(ctx, bad):
    L = Layer(ctx, 10, 5, 6, 40, torch.float32)
    x, xs, h, y, dy = L.T(3), L.R(), L.R(4), L.T(), L.T(5)
    pos = L.pos.clone()
    pos[7] = bad
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.expert_dispatch(L.site, x.t, pos, xs.t)
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.expert_combine(L.site, h.t, L.w, pos, y.t)
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.expert_dispatch_grad(L.site, h.t, pos, y.t)
    with pytest.raises(fb.MapalTrap, match="index_oob"):
        ctx.expert_combine_grad(L.site, h.t, L.w, pos, dy.t, xs.t, torch.empty(10, 5, device="cuda"))
    assert xs.intact() and y.intact() and h.intact()
    ctx.expert_dispatch(L.site, x.t, L.pos, xs.t)  # the flag is clear again


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_stay_in_their_rows(ctx, dtype):
    L = Layer(ctx, 20, 2, 5, 72, dtype)
    h, y = L.R(3), L.T()
    h.t[L.p[4, 1]] = float("nan")
    h.t[L.p[9, 0]] = float("inf")
    h.t[L.there:] = float("nan")  # rows that no slot names are not read
    ctx.expert_combine(L.site, h.t, L.w, L.pos, y.t)
    assert torch.isnan(y.t[4]).all() and not torch.isfinite(y.t[9]).any()
    rest = [t for t in range(20) if t not in (4, 9)]
    assert torch.isfinite(y.t[rest]).all()


def test_a_token_without_experts_gets_zeros(ctx):
    L = Layer(ctx, 6, 2, 4, 33, torch.bfloat16)
    pos = L.pos.clone()
    pos[4:6] = -1
    h, y = L.R(3), L.T()
    y.t.fill_(float("nan"))
    ctx.expert_combine(L.site, h.t, L.w, pos, y.t)
    assert (y.t[2] == 0).all() and torch.isfinite(y.t).all()


def test_no_tokens_and_empty_rows(ctx):
    e = torch.empty(0, dtype=torch.float32, device="cuda")
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    s = fb.expert_site(0, 2, 4, 8, "float32")
    ctx.expert_dispatch(s, e, i, e)
    ctx.expert_combine(s, e, e, i, e)
    ctx.expert_combine_grad(s, e, e, i, e, e, e)
    s = fb.expert_site(3, 2, 4, 0, "float32")
    pos, dw = torch.arange(6, dtype=torch.int32, device="cuda"), torch.ones(6, device="cuda")
    ctx.expert_dispatch(s, e, pos, e)
    ctx.expert_combine(s, e, None, pos, e)
    ctx.expert_combine_grad(s, e, None, pos, e, e, dw)
    assert (dw == 0).all()  # products of no elements


def test_captured_and_replayed(ctx):
    L = Layer(ctx, 64, 4, 16, 512, torch.bfloat16)
    ids, off, pos = random_ids(256, 16, 1), i32(17), i32(256)
    x, xs, y, y2 = L.T(3), L.R(), L.T(), L.T()

    def step():
        ctx.expert_sort(L.site, ids, off, None, pos)
        ctx.expert_dispatch(L.site, x.t, pos, xs.t)
        ctx.expert_combine(L.site, xs.t, L.w, pos, y.t)

    g = replayed(ctx, step)
    ids.copy_(random_ids(256, 16, 99, 0.3))  # other routes in the same graph
    x.t.copy_(randn((64, 512), torch.bfloat16, 98))
    g.replay()
    torch.cuda.synchronize()
    got = y.t.clone()
    xs.t.zero_()
    step()
    assert torch.equal(y.t, got)
    want = (L.w.double() * (pos.view(64, 4) >= 0))[..., None] * x.t.double()[:, None]
    assert_within(y.t, want.sum(1), 5 * U32 * want.abs().sum(1) + out_error(want.sum(1), torch.bfloat16) * 1.01, "y")


def test_offsets_past_32_bits(ctx):
    ld, d = (1 << 30) + 16, 100
    big = torch.as_strided(torch.zeros(5 * ld + d, dtype=torch.int8, device="cuda"), (6, d), (ld, 1))
    site = fb.expert_site(2, 3, 4, d, torch.int8, ldr=ld)
    x = torch.randint(-128, 128, (2, d), device="cuda").to(torch.int8)
    pos = torch.tensor([5, 1, 0, 4, 2, 3], dtype=torch.int32, device="cuda")
    ctx.expert_dispatch(site, x, pos, big)
    assert torch.equal(big, x[[0, 0, 1, 1, 1, 0]])
    big = torch.as_strided(torch.zeros(5 * ld + d, dtype=torch.bfloat16, device="cuda"), (6, d), (ld, 1))
    big.copy_(randn((6, d), torch.bfloat16, 1))
    site = fb.expert_site(2, 3, 4, d, torch.bfloat16, ldr=ld)
    y = torch.empty(2, d, dtype=torch.bfloat16, device="cuda")
    ctx.expert_combine(site, big, None, pos, y)
    want = big.double()[pos.long()].view(2, 3, d).sum(1)
    size = big.double().abs()[pos.long()].view(2, 3, d).sum(1)
    assert_within(y, want, 4 * U32 * size + half_step(torch.bfloat16) * 1.01 * want.abs() + 1e-30, "y")

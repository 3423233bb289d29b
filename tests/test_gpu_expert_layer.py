"""The row-wise operators together, as a layer of experts uses them, on a B200: a serving pass in 8 bits
(norm, rows to 8 bits, sorted by expert with their scales, the experts' products, back with the router's
weights) and a training step in f32 (norm, to the experts and back, every gradient)."""
import pytest
import torch

import flow_b200 as fb
from _rows import U32, assert_within

pytestmark = pytest.mark.gpu


def routed(tokens, k, experts, seed, drop=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    score, ids = torch.topk(torch.randn(tokens, experts, generator=g, device="cuda"), k, dim=1)
    if drop:
        ids[-drop:] = -1
    return ids.to(torch.int32).reshape(-1), torch.softmax(score, 1)


@pytest.mark.parametrize("tokens,k,experts,d,n,drop", [(1, 2, 8, 64, 48, 0), (16, 4, 16, 256, 128, 3), (200, 2, 5, 500, 300, 17),
                                                       (333, 8, 32, 1024, 520, 0)])
def test_serving_pass(tokens, k, experts, d, n, drop):
    with fb.Context((0,), sync=False) as ctx:
        rows = tokens * k
        x = torch.randn(tokens, d, device="cuda").to(torch.bfloat16)
        w, b = torch.randn(d, device="cuda").to(torch.bfloat16), torch.randn(d, device="cuda").to(torch.bfloat16)
        weight = torch.randn(experts, n, d, device="cuda")
        ids, gate = routed(tokens, k, experts, tokens, drop)
        i32 = lambda c: torch.empty(c, dtype=torch.int32, device="cuda")  # noqa: E731
        off, pos = i32(experts + 1), i32(rows)
        normed, y = torch.empty_like(x), torch.empty(tokens, n, dtype=torch.bfloat16, device="cuda")
        q, s = torch.empty(tokens, d, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
        qs, ss = torch.zeros(rows, d, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
        bq, bs = torch.empty(experts, n, d, dtype=torch.int8, device="cuda"), torch.empty(experts, n, device="cuda")
        h = torch.full((rows, n), float("nan"), device="cuda")
        ctx.quantize_rows_i8(fb.quant_site(experts * n, d, "float32"), weight, bq, bs)  # the weights, once

        ctx.layer_norm(fb.norm_site(tokens, d, x.dtype), x, w, b, normed)
        ctx.quantize_rows_i8(fb.quant_site(tokens, d, x.dtype), normed, q, s)
        moved = fb.expert_site(tokens, k, experts, d, torch.int8)
        ctx.expert_sort(moved, ids, off, None, pos)
        ctx.expert_dispatch(moved, q, pos, qs, s, ss)
        ctx.matmul_i8(fb.matmul_i8_site(rows, n, d, h.dtype, groups=experts), qs, ss, bq, bs, h, offsets=off)
        back = fb.expert_site(tokens, k, experts, n, h.dtype)
        out = torch.empty(tokens, n, device="cuda")
        ctx.expert_combine(back, h, gate, pos, out)
        ctx.synchronize()

        # the same from the 8-bit values in f64: exact but for the f32 steps of the scales and the sum
        a = q.double() * s.double()[:, None]
        terms = torch.zeros(tokens, k, n, dtype=torch.float64, device="cuda")
        for e in range(experts):
            t, j = torch.nonzero(ids.view(tokens, k) == e, as_tuple=True)
            terms[t, j] = gate.double()[t, j, None] * (a[t] @ (bq[e].double() * bs[e].double()[:, None]).t())
        assert_within(out, terms.sum(1), (k + 5) * U32 * terms.abs().sum(1), "out")
        # and the whole against the layer without quantising: a row's values are off by half a step of its
        # scale each, so a product of d of them by at most the sum of |weight|*s/2 + |x|*bs/2 + s*bs/4
        real = normed.double()
        worst = torch.zeros(tokens, n, dtype=torch.float64, device="cuda")
        whole = torch.zeros(tokens, n, dtype=torch.float64, device="cuda")
        for e in range(experts):
            t, j = torch.nonzero(ids.view(tokens, k) == e, as_tuple=True)
            g = gate.double()[t, j, None]
            W, B = weight[e].double(), bs[e].double()
            whole.index_add_(0, t, g * (real[t] @ W.t()))
            worst.index_add_(0, t, g * (s.double()[t, None] / 2 * W.abs().sum(1) + real[t].abs().sum(1)[:, None] * B / 2
                                        + d * s.double()[t, None] * B / 4))
        assert_within(out, whole, worst * 1.001 + 1e-6, "out against the layer in f64")


@pytest.mark.parametrize("tokens,k,experts,d,drop", [(5, 2, 4, 33, 0), (120, 3, 9, 260, 11)])
def test_training_step(tokens, k, experts, d, drop):
    """y = combine(scale_e * dispatch(norm(x))), with one scale an expert as its stand-in, and all gradients
    against autograd in f64. Each operator's own error bound is tested in its file; this is about the whole: a
    wrong place, a missing term or weight is off by the entries' own size, while rounding stays at (roundings
    along the path)*2^-24 of the terms, which a row of d entries holds below sqrt(d) times its largest entry
    (their 2-norm), plus 1 for the entries of size 1 that the inputs are drawn with."""
    with fb.Context((0,), sync=False) as ctx:
        rows = tokens * k
        x = torch.randn(tokens, d, device="cuda")
        w, b, dy = torch.randn(d, device="cuda"), torch.randn(d, device="cuda"), torch.randn(tokens, d, device="cuda")
        own = 1 + torch.rand(experts, device="cuda")
        ids, gate = routed(tokens, k, experts, 7, drop)
        i32 = lambda c: torch.zeros(c, dtype=torch.int32, device="cuda")  # noqa: E731
        off, order, pos = i32(experts + 1), i32(rows), i32(rows)
        E = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        ns, es = fb.norm_site(tokens, d, x.dtype), fb.expert_site(tokens, k, experts, d, x.dtype)
        normed, mean, rstd, xs, y = E(tokens, d), E(tokens), E(tokens), E(rows, d), E(tokens, d)
        ctx.layer_norm(ns, x, w, b, normed, mean, rstd)
        ctx.expert_sort(es, ids, off, order, pos)
        ctx.expert_dispatch(es, normed, pos, xs)
        per_row = own[torch.searchsorted(off[1:].contiguous(), torch.arange(rows, device="cuda", dtype=torch.int32),
                                         right=True).clamp(max=experts - 1)]
        h = xs * per_row[:, None]
        ctx.expert_combine(es, h, gate, pos, y)
        dh, dgate, dn, dx, dw, db = E(rows, d), E(tokens, k), E(tokens, d), E(tokens, d), E(d), E(d)
        ctx.expert_combine_grad(es, h, gate, pos, dy, dh, dgate)
        dxs = dh * per_row[:, None]
        ctx.expert_dispatch_grad(es, dxs, pos, dn)
        work = torch.empty(ctx.layer_norm_grad_workspace(ns), dtype=torch.uint8, device="cuda")
        ctx.layer_norm_grad(ns, x, w, mean, rstd, dn, dx, dw, db, work)
        ctx.synchronize()

        X, W, B, G = (t.double().requires_grad_() for t in (x, w, b, gate))
        N = torch.nn.functional.layer_norm(X, (d,), W, B, 1e-5)
        slot = ids.view(tokens, k)
        scale = torch.where(slot >= 0, own.double()[slot.clamp(min=0).long()], 0.0)
        Y = (G * scale).sum(1, keepdim=True) * N
        Y.backward(dy.double())
        for got, want, n in ((y, Y.detach(), 80), (dgate, G.grad, 100), (dx, X.grad, 200), (dw, W.grad, 200 + tokens),
                             (db, B.grad, 100 + tokens)):
            size = want.abs().amax() if want.dim() == 1 else want.abs().amax(1, keepdim=True)
            assert_within(got, want, (n * U32 * (d ** 0.5) * (size + 1)).expand(want.shape), "gradient")


class Served:
    """The serving pass over inputs of its own, its calls on one stream or with the sort on another beside the
    norm and the quantising, joined before the rows move."""

    def __init__(self, tokens, k, experts, d, n, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        bf, rows = torch.bfloat16, tokens * k
        self.x, self.w, self.b = r(tokens, d).to(bf), r(d).to(bf), r(d).to(bf)
        self.ids, self.gate = routed(tokens, k, experts, seed)
        self.bq = torch.randint(-127, 128, (experts, n, d), generator=g, device="cuda").to(torch.int8)
        self.bs = r(experts, n)
        e = lambda *s, t=torch.float32: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
        self.off, self.pos = e(experts + 1, t=torch.int32), e(rows, t=torch.int32)
        self.normed, self.q, self.s = e(tokens, d, t=bf), e(tokens, d, t=torch.int8), e(tokens)
        self.qs, self.ss, self.h, self.out = e(rows, d, t=torch.int8), e(rows), e(rows, n, t=bf), e(tokens, n, t=bf)
        self.ns, self.qsite = fb.norm_site(tokens, d, bf), fb.quant_site(tokens, d, bf)
        self.moved = fb.expert_site(tokens, k, experts, d, torch.int8)
        self.mm = fb.matmul_i8_site(rows, n, d, bf, groups=experts)
        self.back = fb.expert_site(tokens, k, experts, n, bf)

    def run(self, ctx, main, side=None):
        side = side or main
        if side is not main:
            side.wait_stream(main)
        ctx.set_stream(side.cuda_stream)
        ctx.expert_sort(self.moved, self.ids, self.off, None, self.pos)
        ctx.set_stream(main.cuda_stream)
        ctx.layer_norm(self.ns, self.x, self.w, self.b, self.normed)
        ctx.quantize_rows_i8(self.qsite, self.normed, self.q, self.s)
        if side is not main:
            main.wait_stream(side)
        ctx.expert_dispatch(self.moved, self.q, self.pos, self.qs, self.s, self.ss)
        ctx.matmul_i8(self.mm, self.qs, self.ss, self.bq, self.bs, self.h, offsets=self.off)
        ctx.expert_combine(self.back, self.h, self.gate, self.pos, self.out)


@pytest.mark.parametrize("tokens,k,experts,d,n", [(3, 2, 8, 256, 128), (700, 4, 16, 1024, 520)])
@pytest.mark.parametrize("captured", [False, True])
def test_two_streams_that_join(tokens, k, experts, d, n, captured):
    """Sort beside norm on a second stream, joined by an event: run after run in a row, without a wait on the host,
    each over the buffers of the run before, with other inputs, gives what the calls one by one give."""
    with fb.Context((0,), sync=False) as ctx:
        steps = [Served(tokens, k, experts, d, n, i) for i in range(4)]
        main, side = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        want = []
        for s in steps:
            s.run(ctx, main)
            ctx.synchronize()
            want.append(s.out.clone())
        torch.cuda.synchronize()
        s, outs = Served(tokens, k, experts, d, n, 0), [torch.empty_like(want[0]) for _ in range(40)]
        g = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(g, stream=main):
                s.run(ctx, main, side)
        with torch.cuda.stream(main):
            for i, out in enumerate(outs):
                for name in ("x", "w", "b", "ids", "gate", "bq", "bs"):
                    getattr(s, name).copy_(getattr(steps[i % 4], name))
                if captured:
                    g.replay()
                else:
                    s.run(ctx, main, side)
                out.copy_(s.out)
        torch.cuda.synchronize()
        ctx.synchronize()
        for i, out in enumerate(outs):
            assert torch.equal(out, want[i % 4]), f"run {i}"
        del g

"""A training step of a layer of experts as it would be run, forward and backward: norm, tokens sorted by expert, the
experts' products, back, dropout onto the residual, the loss of a vocabulary. Each of the products, dropout and the
loss is held to its formula in f64 on the inputs that the step gave it; the step is the same bits when it is repeated,
captured and replayed."""
import pytest
import torch

import flow_b200 as fb
from _rows import U32, assert_within, out_error, replayed
from test_gpu_dropout import bits
from test_gpu_linear_loss import formula

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = fb.Context((0,))
    yield c
    c.close()


class Step:
    def __init__(self, T=300, k=2, E=5, d=64, n=96, V=1003, p=0.25, t=torch.bfloat16):
        self.T, self.k, self.E, self.d, self.n, self.V, self.p, self.t = T, k, E, d, n, V, p, t
        g = torch.Generator(device="cuda").manual_seed(5)
        r = lambda *s, dtype=t: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
        f = lambda *s, dtype=t: torch.full(s, 7.0, device="cuda").to(dtype)  # noqa: E731
        F, I, rows = torch.float32, torch.int32, T * k
        self.x, self.nw, self.nb = r(T, d), r(d), r(d)
        self.w1, self.w2, self.wv = r(E, n, d) / d ** 0.5, r(E, d, n) / n ** 0.5, r(V, d) / d ** 0.5
        self.gate = torch.softmax(r(T, k, dtype=F), 1).reshape(-1)
        ids = torch.rand(T, E, generator=g, device="cuda").topk(k, 1).indices.to(I)
        ids[T - 40:] = -1  # the padding
        self.ids = ids.reshape(-1)
        self.targets = torch.randint(0, V, (T,), generator=g, device="cuda").to(I)
        self.targets[T - 40:] = -1
        self.rng = torch.tensor([123, 456], device="cuda")
        self.normed, self.mean, self.rstd = f(T, d), f(T, dtype=F), f(T, dtype=F)
        self.offsets, self.pos = f(E + 1, dtype=I), f(rows, dtype=I)
        self.xs, self.h1, self.h2, self.y, self.out = f(rows, d), f(rows, n), f(rows, d), f(T, d), f(T, d)
        self.loss, self.lse, self.g = f(T, dtype=F), f(T, dtype=F), torch.full((T,), 1 / (T - 40), device="cuda")
        self.dout, self.dwv, self.dy = f(T, d), f(V, d), f(T, d)
        self.dh2, self.dgate, self.dh1, self.dw2 = f(rows, d), f(rows, dtype=F), f(rows, n), f(E, d, n)
        self.dxs, self.dw1, self.dn, self.dx = f(rows, d), f(E, n, d), f(T, d), f(T, d)
        self.dnw, self.dnb = f(d, dtype=F), f(d, dtype=F)
        self.OUTS = ("normed offsets pos xs h1 h2 y out loss lse dout dwv dy dh2 dgate dh1 dw2 dxs dw1 dn dx dnw dnb").split()

    def run(self, c):
        T, k, E, d, n, t = self.T, self.k, self.E, self.d, self.n, self.t
        norm, rows = fb.norm_site(T, d, t), fb.expert_site(T, k, E, d, t)
        p1, p2 = fb.product_site(T * k, n, d, t, groups=E), fb.product_site(T * k, d, n, t, groups=E)
        drop, head = fb.dropout_site(T, d, t, self.p), fb.loss_site(T, self.V, d, t)
        if not hasattr(self, "work"):
            self.work = torch.empty(c.linear_loss_workspace(head), dtype=torch.uint8, device="cuda")
            self.nwork = torch.empty(c.layer_norm_grad_workspace(norm), dtype=torch.uint8, device="cuda")
        c.layer_norm(norm, self.x, self.nw, self.nb, self.normed, self.mean, self.rstd)
        c.expert_sort(rows, self.ids, self.offsets, None, self.pos)
        c.expert_dispatch(rows, self.normed, self.pos, self.xs)
        c.product(p1, self.xs, self.w1, self.h1, offsets=self.offsets)
        c.product(p2, self.h1, self.w2, self.h2, offsets=self.offsets)
        c.expert_combine(rows, self.h2, self.gate, self.pos, self.y)
        c.dropout(drop, self.y, self.x, self.out, self.rng)
        c.linear_loss(head, self.out, self.wv, self.targets, self.loss, self.lse, self.work)
        c.linear_loss_grad(head, self.out, self.wv, self.targets, self.lse, self.g, self.dout, self.dwv, self.work)
        c.dropout(drop, self.dout, None, self.dy, self.rng)
        c.expert_combine_grad(rows, self.h2, self.gate, self.pos, self.dy, self.dh2, self.dgate)
        c.product_grad(p2, self.h1, self.w2, self.dh2, self.dh1, self.dw2, offsets=self.offsets)
        c.product_grad(p1, self.xs, self.w1, self.dh1, self.dxs, self.dw1, offsets=self.offsets)
        c.expert_dispatch_grad(rows, self.dxs, self.pos, self.dn)
        c.layer_norm_grad(norm, self.x, self.nw, self.mean, self.rstd, self.dn, self.dx, self.dnw, self.dnb, self.nwork)

    def outs(self):
        return {o: getattr(self, o).clone() for o in self.OUTS}


def check_product(s, x, w, dy, y, dx, dw, what):
    ends, t = s.offsets.tolist(), s.t
    x64, w64, dy64 = x.double(), w.double(), dy.double()
    for g in range(s.E):
        r = slice(ends[g], ends[g + 1])
        for got, a, b, depth in ((y[r], x64[r], w64[g].t(), x.shape[1]), (dx[r], dy64[r], w64[g], w.shape[1]),
                                 (dw[g], dy64[r].t(), x64[r], ends[g + 1] - ends[g])):
            err = (depth + 16) * 17 / 16 * 2 * U32 * (a.abs() @ b.abs())  # as in test_gpu_product.py
            want = a @ b
            assert_within(got, want, err + out_error(want.abs() + err, t), what)
    assert (y[ends[-1]:] == 7).all() and (dx[ends[-1]:] == 7).all()  # rows of no expert


def test_every_operator_on_what_the_step_gave_it(ctx):
    s = Step()
    s.run(ctx)
    o, t = s, s.t
    check_product(s, o.xs, o.w1, o.dh1, o.h1, o.dxs, o.dw1, "first product")
    check_product(s, o.h1, o.w2, o.dh2, o.h2, o.dh1, o.dw2, "second product")
    keep = torch.from_numpy(bits(s.rng, s.T, s.d) >= round(s.p * 65536)).cuda()
    scale = 65536 / (65536 - round(s.p * 65536))
    for got, x, res in ((o.out, o.y, o.x.double()), (o.dy, o.dout, 0.0)):
        want = torch.where(keep, x.double() * scale, 0.0) + res
        assert_within(got, want, out_error(want, t) * (1 + 2 * U32) + 2 * U32 * want.abs() + U32 * x.double().abs() * scale)
    (loss, eloss), (lse, elses), (dh, edh), (dw, edw) = formula(o.out, o.wv, o.targets, o.g, t)[0]
    assert_within(o.loss, loss, eloss, "loss")
    assert_within(o.lse, lse, elses, "lse")
    # the step's own lse goes into its gradient: its error is a relative one of p
    assert_within(o.dout, dh, edh + 2 * elses.max() * (o.g.max() * o.wv.double().abs().sum(0)), "dh")
    assert_within(o.dwv, dw, edw + 2 * elses.max() * (o.g.double() @ o.out.double().abs()), "dw")
    assert not o.dout[s.T - 40:].any() and torch.isfinite(o.dx.float()).all()


def test_repeated_and_captured(ctx):
    s = Step(T=513, k=3, E=7, d=136, n=200, V=2000)
    s.run(ctx)
    first = s.outs()
    for name in s.OUTS:
        getattr(s, name).fill_(7)
    s.run(ctx)
    for name, v in s.outs().items():
        assert torch.equal(v, first[name]), name
    for name in s.OUTS:
        getattr(s, name).fill_(7)
    g = replayed(ctx, lambda: s.run(ctx))
    for name, v in s.outs().items():
        assert torch.equal(v, first[name]), name
    s.rng[1] += 1  # another step's mask, without another capture
    g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(s.out, first["out"]) and torch.equal(s.y, first["y"])


def test_a_captured_step_beside_an_eager_one():
    """Two steps of their own buffers and scratch on two streams, one of them a graph's replays."""
    a, b = Step(), Step(T=200, V=700)
    ca, cb = (fb.Context((0,), sync=False) for _ in range(2))
    a.run(ca)
    b.run(cb)
    torch.cuda.synchronize()
    wa, wb = a.outs(), b.outs()
    g, sa, sb = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=sa):
        ca.set_stream(torch.cuda.current_stream().cuda_stream)
        a.run(ca)
    cb.set_stream(sb.cuda_stream)
    for _ in range(5):
        with torch.cuda.stream(sa):
            g.replay()
        b.run(cb)
    torch.cuda.synchronize()
    assert all(torch.equal(v, wa[n]) for n, v in a.outs().items())
    assert all(torch.equal(v, wb[n]) for n, v in b.outs().items())
    del g
    ca.close()
    cb.close()

"""What the tests of the row-wise operators share: error bounds, guarded buffers, captured calls."""
import torch

U32 = 2.0 ** -24  # half a step of f32, relative
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def out_error(want, dtype):
    """Rounding `want` (f64) once to dtype: half a step, and half the smallest subnormal near zero."""
    f = torch.finfo(dtype)
    return want.abs() * half_step(dtype) + f.smallest_normal * f.eps / 2


def assert_within(got, want, bound, what=""):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    off = (got - want).abs()
    bad = ~nan & ~(off <= bound) & ~(got == want)
    if bad.any():
        i = tuple(int(v[0]) for v in torch.nonzero(bad, as_tuple=True))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: got {got[i].item()!r}, "
                             f"want {want[i].item()!r}, bound {bound[i].item()!r}")


class Guarded:
    """rows x cols at row stride cols + pad, `offset` elements into a buffer filled with a marker: `t` is the
    view, and intact() says whether everything outside it still holds the marker."""

    def __init__(self, rows, cols, dtype, pad=0, offset=0, mark=77):
        ld = cols + pad
        self.rows, self.cols, self.offset, self.ld = rows, cols, offset, ld
        n = offset + rows * ld + 32
        self.buf = torch.full((n,), mark, dtype=dtype, device="cuda")
        self.mark = mark
        self.t = self.buf[offset:offset + rows * ld].view(rows, ld)[:, :cols] if rows and cols else \
            self.buf.new_empty(rows, cols)

    def put(self, values):
        self.t.copy_(values)
        return self

    def intact(self):
        rest = self.buf.clone()
        if self.rows and self.cols:
            rest[self.offset:self.offset + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = self.mark
        return bool((rest == self.mark).all())


def replayed(ctx, fn, times=2):
    """fn captured on a stream of its own through ctx (sync mode off), then replayed."""
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    old = ctx.stream()
    ctx.set_sync(False)
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            fn()
    finally:
        ctx.set_stream(old)
        ctx.set_sync(True)
    for _ in range(times):
        g.replay()
    torch.cuda.synchronize()
    return g

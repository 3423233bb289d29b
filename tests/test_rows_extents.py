"""The row-wise operators take a tensor only if every element that the record says is the tensor's own, without a
GPU: a slice is as long as the slice, however far its storage goes on. CPU tensors on a context object that drives
no device, as in test_rows_refusals.py: an accepted call ends with "ctx is null"."""
import pytest
import torch

import flow_b200 as fb


@pytest.fixture
def ctx():
    c = fb.Context.__new__(fb.Context)
    c._h, c.devices = None, [-1]
    return c


F, I, I8 = torch.float32, torch.int32, torch.int8


def vec(n, dtype=F):
    """n elements and the same again, the caller's own."""
    return torch.zeros(2 * n + 8, dtype=dtype)[:n]


def mat(rows, cols, dtype=F):
    """rows x cols at stride cols + 3 in a longer and wider buffer."""
    return torch.zeros(2 * rows, cols + 3, dtype=dtype)[:rows, :cols]


# method: record, arguments, and which of them are optional
NORM = fb.norm_site(3, 5, F, ldx=8, ldy=8, lddy=8, lddx=8)
EXPERT = fb.expert_site(6, 2, 4, 5, F, ldt=8, ldr=8)
QUANT = fb.quant_site(3, 5, F, ldx=8, ldq=8)
ONE = fb.matmul_i8_site(3, 4, 5, F, lda=8, ldb=8, ldc=7)
MANY = fb.matmul_i8_site(3, 4, 5, F, groups=2, lda=8, ldb=8, ldg=8 * 8, ldc=7)
CALLS = {
    "layer_norm": (NORM, lambda: [mat(3, 5), vec(5), vec(5), mat(3, 5), vec(3), vec(3)], "x w b y mean rstd"),
    "layer_norm_grad": (NORM, lambda: [mat(3, 5), vec(5), vec(3), vec(3), mat(3, 5), mat(3, 5), vec(5), vec(5),
                                       torch.zeros(1 << 12)], "x w mean rstd dy dx dw db"),
    "expert_sort": (EXPERT, lambda: [vec(12, I), vec(5, I), vec(12, I), vec(12, I)], "ids offsets order pos"),
    "expert_dispatch": (EXPERT, lambda: [mat(6, 5), vec(12, I), mat(12, 5), vec(6), vec(12)], "x pos xs scale scale_out"),
    "expert_combine": (EXPERT, lambda: [mat(12, 5), vec(12), vec(12, I), mat(6, 5)], "h w pos y"),
    "expert_dispatch_grad": (EXPERT, lambda: [mat(12, 5), vec(12, I), mat(6, 5)], "dxs pos dx"),
    "expert_combine_grad": (EXPERT, lambda: [mat(12, 5), vec(12), vec(12, I), mat(6, 5), mat(12, 5), vec(12)],
                            "h w pos dy dh dw"),
    "quantize_rows_i8": (QUANT, lambda: [mat(3, 5), mat(3, 5, I8), vec(3)], "x q scale"),
    "matmul_i8": (ONE, lambda: [mat(3, 5, I8), vec(3), mat(4, 5, I8), vec(4), mat(3, 4)], "A scale_a B scale_b C"),
    "matmul_i8 of groups": (MANY, lambda: [mat(3, 5, I8), vec(3), torch.zeros(4, 8, 8, dtype=I8)[:2, :4, :5], vec(8),
                                           mat(3, 4), vec(3, I)], "A scale_a B scale_b C offsets"),
}
ARGUMENTS = [(name, k, what) for name, (_, _, names) in CALLS.items() for k, what in enumerate(names.split())]


def run(ctx, name, args):
    getattr(ctx, name.split()[0])(CALLS[name][0], *args)


@pytest.mark.parametrize("name", CALLS)
def test_slices_of_just_the_records_size_pass(ctx, name):
    with pytest.raises(fb.MapalInfraError, match="ctx is null|not aligned"):
        run(ctx, name, CALLS[name][1]())


def shorter(t):
    """The same buffer with less of it handed over."""
    if t.dim() == 1:
        yield t[:-1]
        yield t[:1]
        yield t[:0]
        yield t[1:]
    elif t.dim() == 2:
        yield t[:-1]
        yield t[1:]
        yield t[:, :-1]
        yield t[:1]
        yield t[:0]
        yield t[:, :0]
        yield torch.zeros(64, 64, dtype=t.dtype).view(-1)[:(t.size(0) - 1) * t.stride(0) + t.size(1) - 1]
    else:
        yield t[:-1]
        yield t[:, :-1]
        yield t[:, :, :-1]
        yield t[:, :, 0]
        yield t[:0]


@pytest.mark.parametrize("name,k,what", ARGUMENTS)
def test_less_than_the_record_is_refused(ctx, name, k, what):
    for i, t in enumerate(shorter(CALLS[name][1]()[k])):
        args = CALLS[name][1]()
        args[k] = t
        with pytest.raises(ValueError, match=f"^{what}"):
            run(ctx, name, args)
            pytest.fail(f"taken: {i}")


@pytest.mark.parametrize("call", [
    lambda c, b, z, i: c.layer_norm(fb.norm_site(3, 5, F), b[:3], None, None, b[:2]),
    lambda c, b, z, i: c.layer_norm(fb.norm_site(3, 5, F, ldy=8), b[:3], None, None, torch.zeros(9, 8)[:, :3]),
    lambda c, b, z, i: c.layer_norm(fb.norm_site(3, 5, F), b[:3], None, None, b[3:6], z[:2]),
    lambda c, b, z, i: c.quantize_rows_i8(fb.quant_site(3, 5, F), b[:3], b[:3].to(I8), z[:1]),
    lambda c, b, z, i: c.expert_sort(fb.expert_site(6, 2, 4, 5, F), i, i[:2], i, i),
    lambda c, b, z, i: c.layer_norm(fb.norm_site(50, 5, F), torch.zeros(50, 5), None, None, torch.zeros(50, 5),
                                    torch.zeros(100)[:3]),
])
def test_slices_with_more_storage_behind_them(ctx, call):
    with pytest.raises(ValueError, match="holds"):
        call(ctx, torch.zeros(10, 5), torch.zeros(10), torch.zeros(12, dtype=I))


@pytest.mark.parametrize("B,ok", [
    (torch.zeros(20, 8, dtype=I8)[:12, :5], True),       # rows of one matrix that holds both groups'
    (torch.zeros(20, 8, dtype=I8)[:11, :5], False),
    (torch.zeros(20, 8, dtype=I8)[:12, :4], False),
    (torch.zeros(96, dtype=I8), True), (torch.zeros(200, dtype=I8)[:92], False), (torch.zeros(200, dtype=I8)[:93], True),
    (torch.zeros(3, 8, 8, dtype=I8)[:, :, :6], True), (torch.zeros(3, 8, 8, dtype=I8)[:1, :, :5], False),
    (torch.zeros(3, 8, 8, dtype=I8)[:2, :3, :5], False),
])
def test_matrices_of_the_products(ctx, B, ok):
    site = fb.matmul_i8_site(3, 4, 5, F, groups=2, ldb=8, ldg=64)
    with pytest.raises(fb.MapalInfraError if ok else ValueError, match="ctx is null|not aligned" if ok else "^B "):
        ctx.matmul_i8(site, torch.zeros(3, 5, dtype=I8), None, B, None, torch.zeros(3, 4), torch.zeros(3, dtype=I))


def test_matrices_between_rows_are_refused(ctx):
    site = fb.matmul_i8_site(3, 2, 3, F, groups=2, ldb=8, ldg=20)  # the second begins inside a row of the view
    with pytest.raises(ValueError, match="not among its rows"):
        ctx.matmul_i8(site, torch.zeros(3, 3, dtype=I8), None, torch.zeros(9, 8, dtype=I8)[:, :7], None,
                      torch.zeros(3, 2), torch.zeros(3, dtype=I))


def test_a_record_of_nothing_takes_any_slice(ctx):
    x = torch.zeros(4, 8)[:, :5]
    with pytest.raises(fb.MapalInfraError, match="ctx is null"):
        ctx.expert_combine(fb.expert_site(3, 2, 4, 5, F, rows=0, ldr=8), x[:, :3], None, torch.zeros(6, dtype=I), torch.zeros(3, 5))


@pytest.mark.parametrize("work", [
    torch.empty(1, dtype=torch.uint8).expand(1 << 20),  # a megabyte by its shape, a byte in memory
    torch.empty(1 << 20)[::2],
    torch.empty(64, 4096)[:, :1024],  # the other columns are the caller's
    torch.empty(64, 64).t()[:32],
])
@pytest.mark.parametrize("direct", [True, False])
def test_scratch_is_contiguous(ctx, work, direct):
    """Through the direct call, which leaves it to the method, and where an address sends the call there at once."""
    x, mean = torch.zeros(3, 5), torch.zeros(3)
    site = fb.norm_site(3, 5, F)
    with pytest.raises(ValueError, match="work must be contiguous"):
        ctx.layer_norm_grad(site, x if direct else x.data_ptr(), None, mean, mean, x, x, torch.zeros(5), None, work)
    with pytest.raises(fb.MapalInfraError, match="ctx is null"):
        ctx.layer_norm_grad(site, x if direct else x.data_ptr(), None, mean, mean, x, x, torch.zeros(5), None,
                            torch.empty(work.shape))

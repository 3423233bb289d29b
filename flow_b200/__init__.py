"""flow_b200 — Python host side of libmapal_gpu, the B200 (sm_100a) runtime
for Mapal's bulk array sites.

The reference's boundary for this path is its CUDA backend: `emit(ir)` turns
each recognized bulk site of a sealed CategoryIr into a kernel plus launch
glue (crates/backends/cuda/src/lib.rs:72-111), and the emitted program
reports a trap with exit code 101 and an infrastructure failure with 102
(module.rs:61-95). Here the kernels are fixed sm_100a kernels behind a C ABI
(include/mapal_gpu.h); this package calls them with the same site records
(TileSite, MoveSite) and maps the ABI's status codes onto exceptions with the
same classes: `MapalTrap` (exit 101: div_zero / index_oob), `Unsupported`
(EmitError::Unsupported) and `MapalInfraError` (exit 102).

Buffers are caller-owned device memory; torch CUDA tensors are accepted as
plain device buffers (torch is plumbing here, never the compute path).
There is no CPU fallback: every call runs a kernel of libmapal_gpu.so.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

from . import _native
from .records import (DTYPES, DropoutSite, ExpertSite, ExprOp, GpuProfile, I8Site, KSplit, LossSite, MoveSite, NormSite,
                      ProductSite, QuantSite, TileRead, TileSite, conv2d_site, dropout_site, expert_site, fir_site,
                      loss_site, matmul_i8_site, matmul_site, norm_site, product_site, program, quant_site,
                      transpose_site)

__all__ = [
    "Context", "MapalTrap", "MapalInfraError", "Unsupported", "TileSite", "TileRead", "KSplit",
    "MoveSite", "GpuProfile", "matmul_site", "fir_site", "conv2d_site", "transpose_site",
    "NormSite", "ExpertSite", "QuantSite", "I8Site", "norm_site", "expert_site", "quant_site", "matmul_i8_site",
    "ProductSite", "LossSite", "DropoutSite", "product_site", "loss_site", "dropout_site",
    "STRICT", "TF32X3", "U11", "U01", "OP_ADD", "OP_SUB", "OP_MUL", "OP_DIV", "OP_MOD",
    "shard_range", "render_f32", "render_f64", "lib",
]

STRICT, TF32X3 = 0, 1
U11, U01 = 0, 1
OP_ADD, OP_SUB, OP_MUL, OP_DIV, OP_MOD = range(5)

OK, TRAP_DIV_ZERO, TRAP_INDEX_OOB = 0, 1, 2
ERR_INVALID, ERR_UNSUPPORTED, ERR_CUDA, ERR_NCCL, ERR_NOMEM, ERR_TIMEOUT = -1, -2, -3, -4, -5, -6


class MapalInfraError(RuntimeError):
    """An infrastructure failure: the reference's exit-102 class (module.rs:66-71)."""
    exit_code = 102

    def __init__(self, status: int, message: str):
        super().__init__(f"[status {status}] {message}")
        self.status = status


class Unsupported(MapalInfraError):
    """A site record this library has no kernel for (EmitError::Unsupported)."""


class MapalTrap(Exception):
    """A defined trap: the reference's exit-101 class (mapal_trap, mapal-rt/src/lib.rs:71-81)."""
    exit_code = 101

    def __init__(self, kind: str):
        super().__init__(f"mapal trap: {kind}")
        self.kind = kind


def lib() -> ctypes.CDLL:
    return _native.load()


def _check(rc: int) -> int:
    if rc == OK:
        return rc
    if rc == TRAP_DIV_ZERO:
        raise MapalTrap("div_zero")
    if rc == TRAP_INDEX_OOB:
        raise MapalTrap("index_oob")
    msg = (lib().mapal_gpu_last_error() or b"").decode(errors="replace")
    if rc == ERR_UNSUPPORTED:
        raise Unsupported(rc, msg)
    raise MapalInfraError(rc, msg)


def _ptr(t) -> int:
    """Address of a buffer: a torch tensor, a numpy array (host), an int address, or None."""
    if t is None:
        return 0
    if isinstance(t, int):
        return t
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    return t.ctypes.data


def _arr(ptrs: Sequence) -> ctypes.Array:
    return (ctypes.c_void_p * len(ptrs))(*[_ptr(p) for p in ptrs])


_SHORT = 1 << 16  # of a direct call: not a status, see binding/rows_py.cpp
_tensor = None  # torch.Tensor, and torch dtypes by MAPAL_DTYPE_* (4: int32, 5: int64), from the first tensor on
_dtypes: list = [None] * 6


class _Direct:
    """The row-wise operators without ctypes (flow_b200/_rows.so, binding/rows_py.cpp): each of its functions takes a
    method's arguments and answers the status, or None for anything but plain tensors that pass the method's checks.
    Bound when the first tensor is checked, since it is built against torch; until then every answer is None."""

    def __init__(self):
        none = lambda *a: None  # noqa: E731
        for name in self.NAMES + self.TRAINING:
            setattr(self, name, none)

    NAMES = ("layer_norm", "layer_norm_grad", "expert_sort", "expert_dispatch", "expert_combine",
             "expert_dispatch_grad", "expert_combine_grad", "quantize_rows_i8", "matmul_i8")
    TRAINING = ("product", "product_grad", "linear_loss", "linear_loss_grad", "dropout")

    def bind(self):
        L = _native.load()
        try:
            from . import _rows
        except ImportError as e:
            raise MapalInfraError(ERR_INVALID, f"flow_b200/_rows.so: {e}; build it with: python -m flow_b200.build") from e
        _rows.bind(tuple(ctypes.cast(getattr(L, "mapal_gpu_" + n), ctypes.c_void_p).value for n in self.NAMES + self.TRAINING),
                   (ctypes.c_void_p, NormSite, ExpertSite, QuantSite, I8Site, ProductSite, LossSite,
                    DropoutSite))
        for name in self.NAMES + self.TRAINING:
            setattr(self, name, getattr(_rows, name))


_direct = _Direct()


def _span(rows: int, cols: int, ld: int) -> int:
    """Elements from the first to the last of rows x cols at row stride ld."""
    return (rows - 1) * ld + cols if rows and cols else 0


def _buf(t, code: int, n: int, device: int, what: str):
    """Address of a device buffer of a row-wise operator: None, an int address taken as given, or a torch tensor,
    which must be of the record's type, on the context's device, contiguous, with `n` elements of its own."""
    if (t.__class__ is _tensor and t.dtype is _dtypes[code] and t.get_device() == device and t.numel() >= n
            and t.is_contiguous()):
        return t.data_ptr()
    return t if t is None else _buf_checked(t, code, n, device, what, 1, n, 0, 1, 0)


def _mat(t, code: int, rows: int, cols: int, ld: int, device: int, what: str, groups: int = 1, ldg: int = 0):
    """The same of rows x cols elements at row stride `ld` (`groups` matrices at `ldg`). A view must lie as the
    record says, whatever dimensions its rows are counted by, and hold all of the record's rows and columns itself:
    what lies behind a slice in its storage is not the call's."""
    need = _span(groups, _span(rows, cols, ld), ldg)
    if (t.__class__ is _tensor and t.dtype is _dtypes[code] and t.get_device() == device and t.numel() >= need
            and t.is_contiguous()):
        return t.data_ptr()
    return t if t is None else _buf_checked(t, code, need, device, what, rows, cols, ld, groups, ldg)


def _buf_checked(t, code: int, need: int, device: int, what: str, rows: int, cols: int, ld: int, groups: int,
                 ldg: int) -> int:
    global _tensor
    if isinstance(t, int):
        return t
    if _tensor is None:
        import torch
        _dtypes[:] = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.int32, torch.int64
        _direct.bind()
        _tensor = torch.Tensor
    if not 0 <= code < len(_dtypes) or t.dtype is not _dtypes[code]:
        raise ValueError(f"{what} is {t.dtype}, the record says {_dtypes[code] if 0 <= code < len(_dtypes) else code}")
    if t.get_device() != device:
        raise ValueError(f"{what} is on {t.device}, the context drives cuda:{device}")
    if not (t.is_contiguous() and t.numel() >= need):
        if t.numel() and t.dim():
            if t.stride(-1) != 1 and t.size(-1) > 1:
                raise ValueError(f"{what}: the elements of a row must be contiguous")
            if not ld and not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous")
            step = ld  # of the dimensions from the last but one on, while they count rows
            for i in range(t.dim() - 2, -1, -1):
                if t.size(i) == 1 or not ld:
                    continue
                if ldg and i == 0 and t.dim() == 3:
                    step = ldg
                if t.stride(i) != step:
                    raise ValueError(f"{what} has row stride {t.stride(i)}, the record says {ld}" if step == ld else
                                     f"{what} has stride {t.stride(i)} in dimension {i}, the record says {step}")
                step *= t.size(i)
        if t.is_contiguous():
            raise ValueError(f"{what} holds {t.numel()} elements, the record needs {need}")
        if need:
            _check_extent(t, what, rows, cols, ld, groups, ldg)
    return t.data_ptr()


def _work(work, dev: int) -> tuple[int, int]:
    """Address and bytes of a scratch tensor of any type."""
    if work is None:
        return 0, 0
    if work.get_device() != dev:
        raise ValueError(f"work is on {work.device}, the context drives cuda:{dev}")
    if not work.is_contiguous():  # its bytes would not be numel() elements in a row
        raise ValueError("work must be contiguous")
    return work.data_ptr(), work.numel() * work.element_size()


def _check_extent(t, what: str, rows: int, cols: int, ld: int, groups: int, ldg: int) -> None:
    """Whether a view of evenly spaced rows holds the record's."""
    if ldg and t.dim() == 3:
        have = t.size(0), t.size(1), t.size(2)
        if have[0] < groups or have[1] < rows or have[2] < cols:
            raise ValueError(f"{what} holds {have[0]} matrices of {have[1]} x {have[2]} elements, the record needs "
                             f"{groups} of {rows} x {cols}")
        return
    if groups > 1:
        if ldg % ld:
            raise ValueError(f"{what}: matrices {ldg} elements apart are not among its rows at stride {ld}")
        rows += (groups - 1) * (ldg // ld)
    have = t.numel() // t.size(-1)
    if have < rows or t.size(-1) < cols:
        raise ValueError(f"{what} holds {have} rows of {t.size(-1)} elements, the record needs {rows} of {cols}")


def _u64s(vals: Sequence[int]) -> ctypes.Array:
    return (ctypes.c_uint64 * len(vals))(*vals)


def shard_range(n: int, nranks: int, r: int) -> tuple[int, int]:
    """[lo, hi) of n units owned by rank r: contiguous, equal up to one unit."""
    lo, hi = ctypes.c_uint64(), ctypes.c_uint64()
    _check(lib().mapal_gpu_shard_range(n, nranks, r, ctypes.byref(lo), ctypes.byref(hi)))
    return lo.value, hi.value


def render_f32(v: float) -> str:
    """Rust `Display` of an f32 (what mapal_print_f32 writes)."""
    buf = ctypes.create_string_buffer(64)
    n = lib().mapal_render_f32(v, buf, 64)
    if n < 0:
        raise MapalInfraError(ERR_INVALID, "render failed")
    return buf.value.decode()


def render_f64(v: float) -> str:
    buf = ctypes.create_string_buffer(400)
    n = lib().mapal_render_f64(v, buf, 400)
    if n < 0:
        raise MapalInfraError(ERR_INVALID, "render failed")
    return buf.value.decode()


def launch_count() -> int:
    """Kernel launches libmapal_gpu has issued in this process so far."""
    return int(lib().mapal_gpu_launch_count())


def nccl_unique_id() -> bytes:
    buf = ctypes.create_string_buffer(128)
    _check(lib().mapal_gpu_nccl_unique_id(buf))
    return buf.raw


class Context:
    """A libmapal_gpu context: streams, trap flags, scratch and (for more than
    one device) NCCL communicators.

    Context(devices=(0,))                       one process, these devices
    Context(devices=(d,), rank=r, nranks=n, nccl_id=id)
                                                one rank of a multi-process job

    With torch_stream=True the library enqueues on torch's current stream of
    each device, so its kernels are ordered with torch work on the same stream.
    """

    def __init__(self, devices: Sequence[int] = (0,), *, rank: int | None = None,
                 nranks: int | None = None, nccl_id: bytes | None = None,
                 torch_stream: bool = True, sync: bool = True):
        L = lib()
        self._h = ctypes.c_void_p()
        self.devices = list(devices)
        if rank is None:
            mask = 0
            for d in self.devices:
                mask |= 1 << d
            _check(L.mapal_gpu_ctx_create(mask, ctypes.byref(self._h)))
        else:
            if len(self.devices) != 1:
                raise ValueError("a rank context drives exactly one device")
            _check(L.mapal_gpu_ctx_create_rank(self.devices[0], nranks, rank, nccl_id,
                                               ctypes.byref(self._h)))
        if torch_stream:
            import torch
            for i, d in enumerate(self.devices):
                s = torch.cuda.current_stream(d)
                _check(L.mapal_gpu_set_stream(self._h, i, ctypes.c_void_p(s.cuda_stream)))
        self.set_sync(sync)

    # ---- lifecycle -------------------------------------------------------------
    def close(self) -> None:
        if self._h:
            lib().mapal_gpu_ctx_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __enter__(self) -> "Context":
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def profile(self, local: int = 0) -> GpuProfile:
        p = GpuProfile()
        _check(lib().mapal_gpu_profile(self._h, local, ctypes.byref(p)))
        return p

    def world(self) -> tuple[int, int]:
        n, r = ctypes.c_int(), ctypes.c_int()
        _check(lib().mapal_gpu_ctx_world(self._h, ctypes.byref(n), ctypes.byref(r)))
        return n.value, r.value

    def sum_combine(self) -> int:
        """1: sharded sums combine over peer memory; -1: NCCL all-reduce; 0: not yet decided."""
        m = ctypes.c_int()
        _check(lib().mapal_gpu_ctx_sum_combine(self._h, ctypes.byref(m)))
        return m.value

    def stream(self, local: int = 0) -> int:
        s = ctypes.c_void_p()
        _check(lib().mapal_gpu_get_stream(self._h, local, ctypes.byref(s)))
        return s.value or 0

    def set_stream(self, stream: int | None, local: int = 0) -> None:
        _check(lib().mapal_gpu_set_stream(self._h, local, ctypes.c_void_p(stream or 0)))

    def set_sync(self, sync: bool) -> None:
        _check(lib().mapal_gpu_set_sync(self._h, 1 if sync else 0))

    def synchronize(self) -> None:
        _check(lib().mapal_gpu_synchronize(self._h))

    # ---- generators --------------------------------------------------------------
    def iota(self, out) -> None:
        _check(lib().mapal_gpu_iota_i32(self._h, _ptr(out), out.numel()))

    def fill(self, out, v: float) -> None:
        _check(lib().mapal_gpu_fill_f32(self._h, _ptr(out), v, out.numel()))

    def widen(self, inp, out) -> None:
        _check(lib().mapal_gpu_widen_i32_f32(self._h, _ptr(inp), _ptr(out), out.numel()))

    def gen_affine(self, out, mul: int, add: int, mod: int, sub: int, start: int = 0) -> None:
        _check(lib().mapal_gpu_gen_affine_f32(self._h, _ptr(out), out.numel(), start, mul, add, mod, sub))

    def gen(self, out, seed: int, offset: int = 0, kind: int = U11) -> None:
        _check(lib().mapal_gpu_gen_f32(self._h, _ptr(out), out.numel(), seed, offset, kind))

    def gen_index(self, out, seed: int, offset: int, rng: int) -> None:
        _check(lib().mapal_gpu_gen_index_i32(self._h, _ptr(out), out.numel(), seed, offset, rng))

    # ---- sites ----------------------------------------------------------------------
    def saxpy(self, a: float, x, y0, out) -> None:
        _check(lib().mapal_gpu_map_saxpy(self._h, a, _ptr(x), _ptr(y0), _ptr(out), out.numel()))

    def zip_map(self, op: int, x, y, out) -> None:
        _check(lib().mapal_gpu_zip_map_f32(self._h, op, _ptr(x), _ptr(y), _ptr(out), out.numel()))

    def map_expr(self, prog, arrays, out, n: int | None = None) -> None:
        """out[t] = prog evaluated at element t (see records.program)."""
        n = out.numel() if n is None else n
        lens = _u64s([a.numel() for a in arrays]) if arrays else None
        _check(lib().mapal_gpu_map_expr(self._h, prog, len(prog), _arr(arrays) if arrays else None, lens,
                                        len(arrays), _ptr(out), n))

    def transpose(self, site: MoveSite, inp, out) -> None:
        _check(lib().mapal_gpu_transpose(self._h, ctypes.byref(site), _ptr(inp), _ptr(out)))

    def gather(self, x, idx, out) -> None:
        _check(lib().mapal_gpu_gather(self._h, _ptr(x), x.numel(), _ptr(idx), _ptr(out), out.numel()))

    def fold_sum(self, x, out, seed: float = 0.0) -> None:
        """out (one device float) = seed + sum(x), tree order, f64 accumulation."""
        _check(lib().mapal_gpu_fold_sum_f32(self._h, seed, _ptr(x), x.numel(), _ptr(out)))

    def fold_sum_i32(self, x, out, seed: int = 0) -> None:
        """out (one device int32) = seed + sum(x) with wrapping i32 arithmetic (exact in any order)."""
        _check(lib().mapal_gpu_fold_sum_i32(self._h, seed, _ptr(x), x.numel(), _ptr(out)))

    def fold_sum_strict(self, x, out, seed: float = 0.0) -> None:
        """out (one device float) = the interpreter's left fold of x from seed, bit-exact."""
        _check(lib().mapal_gpu_fold_sum_f32_strict(self._h, seed, _ptr(x), x.numel(), _ptr(out)))

    def fir(self, site: TileSite, w, x, out) -> None:
        _check(lib().mapal_gpu_fir_f32(self._h, ctypes.byref(site), _ptr(w), _ptr(x), _ptr(out)))

    def conv2d_3x3(self, site: TileSite, w, img, out) -> None:
        _check(lib().mapal_gpu_conv2d_3x3_f32(self._h, ctypes.byref(site), _ptr(w), _ptr(img), _ptr(out)))

    def matmul(self, site: TileSite, A, B, C, mode: int = STRICT) -> None:
        _check(lib().mapal_gpu_matmul_f32(self._h, ctypes.byref(site), _ptr(A), _ptr(B), _ptr(C), mode))

    def matmul_host(self, site: TileSite, A, B, C, mode: int = STRICT) -> None:
        """The matmul site on HOST buffers (torch CPU tensors, pinned for overlap, or
        numpy arrays): copies in, multiply and copy out overlap in row blocks."""
        _check(lib().mapal_gpu_matmul_f32_host(self._h, ctypes.byref(site), _ptr(A), _ptr(B), _ptr(C), mode))

    def matmul_host_sharded(self, site: TileSite, As, Bs, Cs, rows: Sequence[int], mode: int = STRICT) -> None:
        """The host-array matmul over the context's ranks: As[d] / Cs[d] are the local
        device's row blocks in host memory, Bs[d] a host copy of the whole B."""
        _check(lib().mapal_gpu_matmul_f32_host_sharded(self._h, ctypes.byref(site), _arr(As), _arr(Bs), _arr(Cs),
                                                       _u64s(rows), mode))

    def tile_site(self, site: TileSite, a, b, out, mode: int = STRICT) -> None:
        _check(lib().mapal_gpu_tile_site_f32(self._h, ctypes.byref(site), _ptr(a), _ptr(b), _ptr(out), mode))

    # ---- rows of a model's layer (local device 0) --------------------------------------
    def layer_norm(self, site: NormSite, x, w, b, y, mean=None, rstd=None) -> None:
        """y = (x - mean(x)) / sqrt(var(x) + eps) * w + b for each row; mean and rstd for the gradient."""
        rc = _direct.layer_norm(self._h, self.devices[0], site, x, w, b, y, mean, rstd)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, rows, d, t, ldx, ldy = self.devices[0], site.rows, site.d, site.dtype, site.ldx, site.ldy
        _check(_native.load().mapal_gpu_layer_norm(
            self._h, site, _mat(x, t, rows, d, ldx, dev, "x"),
            _buf(w, site.wtype, d, dev, "w"), _buf(b, site.wtype, d, dev, "b"),
            _mat(y, t, rows, d, ldy, dev, "y"), _buf(mean, 0, rows, dev, "mean"),
            _buf(rstd, 0, rows, dev, "rstd")))

    def layer_norm_grad_workspace(self, site: NormSite) -> int:
        """Bytes of scratch that layer_norm_grad takes."""
        n = ctypes.c_uint64()
        _check(_native.load().mapal_gpu_layer_norm_grad_workspace(self._h, site, ctypes.byref(n)))
        return n.value

    def layer_norm_grad(self, site: NormSite, x, w, mean, rstd, dy, dx, dw, db, work) -> None:
        """dx, dw and db (f32; either may be None) of layer_norm. `work`: a contiguous CUDA buffer of at least
        layer_norm_grad_workspace(site) bytes, its own for calls that may overlap."""
        rc = _direct.layer_norm_grad(self._h, self.devices[0], site, x, w, mean, rstd, dy, dx, dw, db, work)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, rows, d, t = self.devices[0], site.rows, site.d, site.dtype
        at, n = _work(work, dev)
        _check(_native.load().mapal_gpu_layer_norm_grad(
            self._h, site, _mat(x, t, rows, d, site.ldx, dev, "x"),
            _buf(w, site.wtype, d, dev, "w"), _buf(mean, 0, rows, dev, "mean"), _buf(rstd, 0, rows, dev, "rstd"),
            _mat(dy, t, rows, d, site.lddy, dev, "dy"),
            _mat(dx, t, rows, d, site.lddx, dev, "dx"), _buf(dw, 0, d, dev, "dw"),
            _buf(db, 0, d, dev, "db"), at, n))

    def expert_sort(self, site: ExpertSite, ids, offsets, order, pos) -> None:
        """Slots sorted by expert, stably: offsets (experts + 1), order (place -> slot; may be None) and pos
        (slot -> place, -1 where ids is -1), all int32."""
        rc = _direct.expert_sort(self._h, self.devices[0], site, ids, offsets, order, pos)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, n = self.devices[0], site.tokens * site.k
        _check(_native.load().mapal_gpu_expert_sort(
            self._h, site, _buf(ids, 4, n, dev, "ids"),
            _buf(offsets, 4, site.experts + 1, dev, "offsets"), _buf(order, 4, n, dev, "order"),
            _buf(pos, 4, n, dev, "pos")))

    def expert_dispatch(self, site: ExpertSite, x, pos, xs, scale=None, scale_out=None) -> None:
        """xs[pos[t, j]] = x[t], and scale_out likewise from scale (the scales of 8-bit rows)."""
        rc = _direct.expert_dispatch(self._h, self.devices[0], site, x, pos, xs, scale, scale_out)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, t, d, tokens = self.devices[0], site.dtype, site.d, site.tokens
        _check(_native.load().mapal_gpu_expert_dispatch(
            self._h, site, _mat(x, t, tokens, d, site.ldt, dev, "x"),
            _buf(scale, 0, tokens, dev, "scale"), _buf(pos, 4, tokens * site.k, dev, "pos"),
            _mat(xs, t, site.rows, d, site.ldr, dev, "xs"),
            _buf(scale_out, 0, site.rows, dev, "scale_out")))

    def expert_combine(self, site: ExpertSite, h, w, pos, y) -> None:
        """y[t] = sum over j of w[t, j] * h[pos[t, j]] (w None: 1)."""
        rc = _direct.expert_combine(self._h, self.devices[0], site, h, w, pos, y)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, t, d, tokens = self.devices[0], site.dtype, site.d, site.tokens
        _check(_native.load().mapal_gpu_expert_combine(
            self._h, site, _mat(h, t, site.rows, d, site.ldr, dev, "h"),
            _buf(w, 0, tokens * site.k, dev, "w"), _buf(pos, 4, tokens * site.k, dev, "pos"),
            _mat(y, t, tokens, d, site.ldt, dev, "y")))

    def expert_dispatch_grad(self, site: ExpertSite, dxs, pos, dx) -> None:
        """dx[t] = sum over j of dxs[pos[t, j]]."""
        rc = _direct.expert_dispatch_grad(self._h, self.devices[0], site, dxs, pos, dx)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, t, d, tokens = self.devices[0], site.dtype, site.d, site.tokens
        _check(_native.load().mapal_gpu_expert_dispatch_grad(
            self._h, site, _mat(dxs, t, site.rows, d, site.ldr, dev, "dxs"),
            _buf(pos, 4, tokens * site.k, dev, "pos"), _mat(dx, t, tokens, d, site.ldt, dev, "dx")))

    def expert_combine_grad(self, site: ExpertSite, h, w, pos, dy, dh, dw) -> None:
        """dh[pos[t, j]] = w[t, j] * dy[t] and dw[t, j] = <dy[t], h[pos[t, j]]> (dw may be None)."""
        rc = _direct.expert_combine_grad(self._h, self.devices[0], site, h, w, pos, dy, dh, dw)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, t, d, tokens, n = self.devices[0], site.dtype, site.d, site.tokens, site.tokens * site.k
        _check(_native.load().mapal_gpu_expert_combine_grad(
            self._h, site, _mat(h, t, site.rows, d, site.ldr, dev, "h"), _buf(w, 0, n, dev, "w"),
            _buf(pos, 4, n, dev, "pos"), _mat(dy, t, tokens, d, site.ldt, dev, "dy"),
            _mat(dh, t, site.rows, d, site.ldr, dev, "dh"), _buf(dw, 0, n, dev, "dw")))

    def quantize_rows_i8(self, site: QuantSite, x, q, scale) -> None:
        """scale = max|x|/127 and q = x/scale rounded to int8, for each row."""
        rc = _direct.quantize_rows_i8(self._h, self.devices[0], site, x, q, scale)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, rows, d = self.devices[0], site.rows, site.d
        _check(_native.load().mapal_gpu_quantize_rows_i8(
            self._h, site, _mat(x, site.dtype, rows, d, site.ldx, dev, "x"),
            _mat(q, 3, rows, d, site.ldq, dev, "q"), _buf(scale, 0, rows, dev, "scale")))

    def matmul_i8(self, site: I8Site, A, scale_a, B, scale_b, C, offsets=None) -> None:
        """C[i] = (A[i] . B[g]^T) * scale_a[i] * scale_b[g] with exact integer sums; rows offsets[g] to
        offsets[g + 1] belong to g (offsets None: one matrix for all rows)."""
        rc = _direct.matmul_i8(self._h, self.devices[0], site, A, scale_a, B, scale_b, C, offsets)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, m, n, k, groups, ldb = self.devices[0], site.m, site.n, site.k, site.groups, site.ldb
        _check(_native.load().mapal_gpu_matmul_i8(
            self._h, site, _mat(A, 3, m, k, site.lda, dev, "A"),
            _buf(scale_a, 0, m, dev, "scale_a"),
            _mat(B, 3, n, k, ldb, dev, "B", groups, site.ldg),
            _buf(scale_b, 0, groups * n, dev, "scale_b"), _buf(offsets, 4, groups + 1, dev, "offsets"),
            _mat(C, site.dtype, m, n, site.ldc, dev, "C")))

    def product(self, site: ProductSite, x, w, y, offsets=None) -> None:
        """y[i] = w[g] . x[i] in 16-bit floats with f32 sums; rows offsets[g] to offsets[g + 1] belong to g (offsets
        None: one matrix for all rows)."""
        rc = _direct.product(self._h, self.devices[0], site, x, w, y, offsets)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, m, n, k, groups, t = self.devices[0], site.m, site.n, site.k, site.groups, site.dtype
        _check(_native.load().mapal_gpu_product(
            self._h, site, _mat(x, t, m, k, site.ldx, dev, "x"), _mat(w, t, n, k, site.ldw, dev, "w", groups, site.ldg),
            _buf(offsets, 4, groups + 1, dev, "offsets"), _mat(y, site.ytype, m, n, site.ldy, dev, "y")))

    def product_grad(self, site: ProductSite, x, w, dy, dx, dw, offsets=None) -> None:
        """dx[i] = w[g]^T . dy[i] and dw[g] = the sum over g's rows of dy[i]^T . x[i]; either may be None."""
        rc = _direct.product_grad(self._h, self.devices[0], site, x, w, dy, dx, dw, offsets)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, m, n, k, groups, t = self.devices[0], site.m, site.n, site.k, site.groups, site.dtype
        _check(_native.load().mapal_gpu_product_grad(
            self._h, site, _mat(x, t, m, k, site.ldx, dev, "x"), _mat(w, t, n, k, site.ldw, dev, "w", groups, site.ldg),
            _buf(offsets, 4, groups + 1, dev, "offsets"), _mat(dy, t, m, n, site.lddy, dev, "dy"),
            _mat(dx, t, m, k, site.lddx, dev, "dx"), _mat(dw, site.dwtype, n, k, site.lddw, dev, "dw", groups, site.lddg)))

    def linear_loss_workspace(self, site: LossSite, w=None, grad: bool = True) -> int:
        """Bytes of scratch that linear_loss takes, or (grad) that serve its gradient too. `w`: the weights that the
        calls will be given, where they may lie off a 16-byte boundary."""
        n = ctypes.c_uint64()
        _check(_native.load().mapal_gpu_linear_loss_workspace(self._h, site, _ptr(w), 1 if grad else 0, ctypes.byref(n)))
        return n.value

    def linear_loss(self, site: LossSite, h, w, targets, loss, lse, work) -> None:
        """loss[i] = lse[i] - <h[i], w[targets[i]]> with lse[i] the log of the summed exponentials of <h[i], w[v]> over
        the vocabulary, both f32; a row whose target is -1 has a loss of 0. lse may be None, and rows without a target
        are then not read. `work`: a contiguous CUDA buffer of at least linear_loss_workspace(site) bytes, its own for
        calls that may overlap."""
        rc = _direct.linear_loss(self._h, self.devices[0], site, h, w, targets, loss, lse, work)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, rows, vocab, d, t = self.devices[0], site.rows, site.vocab, site.d, site.dtype
        at, n = _work(work, dev)
        _check(_native.load().mapal_gpu_linear_loss(
            self._h, site, _mat(h, t, rows, d, site.ldh, dev, "h"), _mat(w, t, vocab, d, site.ldw, dev, "w"),
            _buf(targets, 4, rows, dev, "targets"), _buf(loss, 0, rows, dev, "loss"), _buf(lse, 0, rows, dev, "lse"),
            at, n))

    def linear_loss_grad(self, site: LossSite, h, w, targets, lse, dloss, dh, dw, work) -> None:
        """dh and dw (either may be None) of linear_loss from its lse and the loss's gradient, one f32 a row (None:
        1)."""
        rc = _direct.linear_loss_grad(self._h, self.devices[0], site, h, w, targets, lse, dloss, dh, dw, work)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, rows, vocab, d, t = self.devices[0], site.rows, site.vocab, site.d, site.dtype
        at, n = _work(work, dev)
        _check(_native.load().mapal_gpu_linear_loss_grad(
            self._h, site, _mat(h, t, rows, d, site.ldh, dev, "h"), _mat(w, t, vocab, d, site.ldw, dev, "w"),
            _buf(targets, 4, rows, dev, "targets"), _buf(lse, 0, rows, dev, "lse"),
            _buf(dloss, 0, rows, dev, "dloss"), _mat(dh, t, rows, d, site.lddh, dev, "dh"),
            _mat(dw, t, vocab, d, site.lddw, dev, "dw"), at, n))

    def dropout(self, site: DropoutSite, x, residual, y, rng) -> None:
        """y = residual + x/(1 - p) where the generator keeps the element, residual alone elsewhere (residual None: 0).
        `rng`: two int64 on the device, the key and the place in its stream; a call's mask depends on these, the row
        and the column alone, so the gradient is the same call on dy without a residual."""
        rc = _direct.dropout(self._h, self.devices[0], site, x, residual, y, rng)
        if rc is not None and rc != _SHORT:
            if rc:
                _check(rc)
            return
        dev, rows, d, t = self.devices[0], site.rows, site.d, site.dtype
        _check(_native.load().mapal_gpu_dropout(
            self._h, site, _mat(x, t, rows, d, site.ldx, dev, "x"), _mat(residual, t, rows, d, site.ldr, dev, "residual"),
            _buf(rng, 5, 2, dev, "rng"), _mat(y, t, rows, d, site.ldy, dev, "y")))

    # ---- sharded sites (one buffer per local device) --------------------------------
    def saxpy_sharded(self, a: float, xs, y0s, outs) -> None:
        n = _u64s([o.numel() for o in outs])
        _check(lib().mapal_gpu_saxpy_sharded(self._h, a, _arr(xs), _arr(y0s), _arr(outs), n))

    def fold_sum_sharded(self, xs, outs, seed: float = 0.0) -> None:
        n = _u64s([x.numel() for x in xs])
        _check(lib().mapal_gpu_fold_sum_f32_sharded(self._h, seed, _arr(xs), n, _arr(outs)))

    def broadcast(self, bufs, root: int = 0) -> None:
        _check(lib().mapal_gpu_broadcast_f32(self._h, _arr(bufs), bufs[0].numel(), root))

    def gather_sharded(self, xs, idxs, outs) -> None:
        n = _u64s([o.numel() for o in outs])
        _check(lib().mapal_gpu_gather_sharded(self._h, _arr(xs), xs[0].numel(), _arr(idxs), _arr(outs), n))

    def probe_mma_peak(self, kind: int = 0, iters: int = 4096) -> float:
        """Measured tensor-pipe rate in TFLOP/s of the 3xTF32 GEMM's MMA shape
        (kind 0: tf32; kind 1: the bf16 form of the same shape), operands
        resident in shared memory, one CTA per SM."""
        out = ctypes.c_double()
        _check(lib().mapal_gpu_probe_mma_peak(self._h, kind, iters, ctypes.byref(out)))
        return out.value

    def probe_launch_floor(self, kind: int, x=None, sink=None) -> None:
        """Enqueue the floor kernel: kind 0 an empty kernel, kind 1 a read of
        x with the sum fold's grid and loads but no combine."""
        n = x.numel() if x is not None else 0
        _check(lib().mapal_gpu_probe_launch_floor(self._h, kind, _ptr(x) if x is not None else None, n,
                                                  _ptr(sink) if sink is not None else None))

    def matmul_sharded(self, site: TileSite, As, Bs, Cs, rows: Sequence[int], root: int = 0,
                       mode: int = STRICT) -> None:
        _check(lib().mapal_gpu_matmul_f32_sharded(self._h, ctypes.byref(site), _arr(As), _arr(Bs),
                                                  _arr(Cs), _u64s(rows), root, mode))


def device_count() -> int:
    n = ctypes.c_int()
    _check(lib().mapal_gpu_device_count(ctypes.byref(n)))
    return n.value

// product.cu — products in 16-bit floats with one matrix or one per group of rows,
// and their gradients (mapal_gpu_product*). No counterpart in the reference.
#include "product.cuh"

namespace cg = cooperative_groups;

namespace {

// ---- any operands ----------------------------------------------------------------------
//
// One CTA a tile of 128 lanes by NT columns. Copying warps bring a block of t at
// a time into the swizzled layout of shared memory, from operands at any place and
// stride: both layouts are lines of 128 bytes (a K-major line is a lane's or
// column's 64 steps of t, an MN-major one 64 lanes or columns at one step), so
// one loop serves all three products. Steps behind the group's last are zeros in
// both operands.

constexpr int kCopyThreads = 512;
constexpr int kAnyOut = 4;  // warps that write

template <int NT, int STAGES>
struct AnySmem {
  uint8_t stage[STAGES][(128 + NT) * 128];  // A's lines, then B's
  uint64_t full[STAGES], empty[STAGES];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drained;
  uint32_t tmem_base;
  int abort;
};

struct AnyOperand {
  const uint8_t* base;
  uint64_t ld, ldg;  // bytes
};

// A thread's share of one operand's block: 16 bytes of every kCopyThreads/8-th line.
template <bool MN, int LINES>
struct Lines {
  static constexpr int kTurns = (LINES * 8 + kCopyThreads - 1) / kCopyThreads;
  const uint8_t* at;  // this thread's 16 bytes of its first line, at the block's t
  uint64_t step;      // to its next line
  uint64_t ld;
  int32_t rows;   // K-major: lines that exist; MN-major: steps of t that are left
  int32_t width;  // elements from this thread's first on: K-major of t, MN-major of lanes or columns
  uint4 a[kTurns], b[kTurns];

  // first: the address of (first lane or column, first step of t).
  __device__ __forceinline__ void set(const uint8_t* first, uint64_t ld_, uint32_t extent, uint32_t depth) {
    const uint32_t c = threadIdx.x & 7, line = threadIdx.x >> 3;
    ld = ld_;
    at = first + line * ld_ + c * 16;
    step = kCopyThreads / 8 * ld_;
    if (MN) {
      rows = (int32_t)min(depth, 0x7fffffffu);
      width = (int32_t)extent - (int32_t)(c * 8);
      // lines 64.. are the next 64 lanes or columns at the same steps
    } else {
      rows = (int32_t)extent;
      width = (int32_t)min(depth, 0x7fffffffu) - (int32_t)(c * 8);
    }
  }
  static_assert(kCopyThreads / 8 == kStepK, "a turn is one 64 lines: an MN-major chunk");

  // Elements of the 16 bytes of turn i that exist, 0 to 8.
  __device__ __forceinline__ int have(int i) const {
    const int line = (int)(threadIdx.x >> 3);
    const bool there = (MN ? line : line + i * (kCopyThreads / 8)) < rows && (LINES >= kCopyThreads / 8 || line < LINES);
    const int w = MN ? width - i * 64 : width;
    return there ? max(0, min(8, w)) : 0;
  }
  __device__ __forceinline__ const uint8_t* place(int i) const { return MN ? at + i * 128 : at + i * step; }

  // The aligned words that hold the elements: none is read without one of them.
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int n = have(i);
      const uint8_t* p = place(i);
      const uint32_t sh = (uint32_t)(uintptr_t)p & 15;
      const uint4* w = reinterpret_cast<const uint4*>(p - sh);
      a[i] = n > 0 ? __ldg(w) : make_uint4(0, 0, 0, 0);
      b[i] = n > 0 && sh + 2 * n > 16 ? __ldg(w + 1) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void store(uint8_t* tile) const {
    const uint32_t c = threadIdx.x & 7, line = threadIdx.x >> 3;
    if (LINES < kCopyThreads / 8 && line >= LINES) return;
    uint8_t* to = tile + line * 128 + ((c ^ (line & 7)) << 4);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int n = have(i);
      uint4 v = straddle(a[i], b[i], (uint32_t)(uintptr_t)place(i) & 15);
      if (n < 8) {
        uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = n >= 2 * k + 2 ? q[k] : n == 2 * k + 1 ? q[k] & 0xffffu : 0u;
        v = make_uint4(q[0], q[1], q[2], q[3]);
      }
      *reinterpret_cast<uint4*>(to + i * (kStepK * 128)) = v;
    }
  }
  __device__ __forceinline__ void next() {
    if (MN) {
      at += kStepK * ld;
      rows -= kStepK;
    } else {
      at += 128;
      width -= kStepK;
    }
  }
};

template <int MODE, typename T, int NT, int STAGES>
__global__ void __launch_bounds__(kCopyThreads + 32 * (1 + kAnyOut), 1)
    product_any_kernel(const AnyOperand A, const AnyOperand B, const __grid_constant__ ProductArgs P,
                       const StoreTile<MODE, T> out) {
  using Smem = AnySmem<NT, STAGES>;
  constexpr uint32_t kCols = 2 * NT;
  constexpr int kCopy = kCopyThreads / 32;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  volatile int* abort = &sm.abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sm.full[s], kCopyThreads);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], kAnyOut);
    }
    mbar_init(&sm.drained, 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  grid_wait();
  grid_go();
  if (warp == kCopy) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(&sm.tmem_base)),
                 "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;
  JobWalk<MODE> walk(P, NT, 128);
  Job j;
  bool more = walk.at(blockIdx.x, j);
  uint32_t it = 0;

  if (warp < kCopy) {
    // ---- copies ----
    Lines<MODE != kForward, 128> la;
    Lines<MODE == kGradW, NT> lb;
    for (uint64_t tile = blockIdx.x; more; tile += gridDim.x, more = walk.at(tile, j)) {
      // (lane, t) and (col, t) of the operands: K-major ones run along t
      const uint8_t* a = A.base + (MODE == kGradW ? 0 : j.group * A.ldg);
      a += MODE == kForward ? j.lane0 * A.ld + 2ull * j.t0 : j.t0 * A.ld + 2ull * j.lane0;
      const uint8_t* b = B.base + (MODE == kGradW ? j.t0 * B.ld + 2ull * j.col0 : j.col0 * B.ld + 2ull * j.t0);
      la.set(a, A.ld, P.lanes - j.lane0, j.depth);
      lb.set(b, B.ld, j.cols, j.depth);
      const uint32_t blocks = (j.depth + kStepK - 1) / kStepK;
      bool gone = false;
      if (blocks) {
        la.load();
        lb.load();
      }
#pragma unroll 1
      for (uint32_t kb = 0; kb < blocks; ++kb, ++it) {
        const uint32_t s = it % STAGES;
        gone = any_of(!mbar_wait(&sm.empty[s], ((it / STAGES) & 1) ^ 1, abort));
        if (gone) break;
        la.store(sm.stage[s]);
        lb.store(sm.stage[s] + 128 * 128);
        if (kb + 1 < blocks) {  // the next block's loads run beside this one's products
          la.next();
          lb.next();
          la.load();
          lb.load();
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&sm.full[s]);
      }
      if (gone) *abort = 1;
      if (any_of(*abort)) break;
    }
  } else if (warp == kCopy) {
    // ---- products ----
    uint32_t n = 0;
    for (uint64_t tile = blockIdx.x; more; tile += gridDim.x, more = walk.at(tile, j), ++n) {
      const uint32_t b = n & 1, blocks = (j.depth + kStepK - 1) / kStepK;
      if (elect_one()) {
        const uint32_t idesc = idesc_f16<MODE>(P.bf16, 128, (int)((j.cols + 15) / 16 * 16));
        if (!mbar_wait(&sm.acc_empty[b], ((n >> 1) & 1) ^ 1, abort)) *abort = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (uint32_t kb = 0; kb < blocks && !*abort; ++kb, ++it) {
          const uint32_t s = it % STAGES;
          if (!mbar_wait(&sm.full[s], (it / STAGES) & 1, abort)) {
            *abort = 1;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = operand_desc<MODE != kForward>(sm.stage[s]),
                         db = operand_desc<MODE == kGradW>(sm.stage[s] + 128 * 128);
#pragma unroll
          for (uint32_t kk = 0; kk < kStepK / 16; ++kk)
            mma_f16<1>(tmem + b * NT, da + kk * operand_step<MODE != kForward>(),
                       db + kk * operand_step<MODE == kGradW>(), idesc, kb > 0 || kk > 0);
          mma_commit(&sm.empty[s]);
        }
        mma_commit(&sm.acc_full[b]);
      }
      if (any_of(*abort)) break;
    }
  } else {
    // ---- output ----
    const int quarter = warp & 3;
    uint32_t n = 0;
    for (uint64_t tile = blockIdx.x; more; tile += gridDim.x, more = walk.at(tile, j), ++n) {
      const uint32_t b = n & 1;
      if (any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort)) {
        *abort = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      out.put(P, j, tmem + ((uint32_t)(quarter * 32) << 16) + b * NT, j.lane0 + quarter * 32 + lane, 0, NT);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort) {
    if (threadIdx.x == 0) atomicOr(P.trap, kDeviceTimeout);
    if (warp == kCopy && elect_one()) {
      mma_commit(&sm.drained);
      mbar_wait(&sm.drained, 0, nullptr);
    }
    __syncthreads();
  }
  if (warp == kCopy) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
  }
}

// ---- host ------------------------------------------------------------------------------

template <int MODE, typename T, int NT, int STAGES>
int launch_any(const DeviceSlot& D, const Operands& o, const ProductArgs& P, const StoreTile<MODE, T>& out) {
  constexpr size_t smem = sizeof(AnySmem<NT, STAGES>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  auto kernel = product_any_kernel<MODE, T, NT, STAGES>;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, smem, "product shared memory"));
  const AnyOperand A{static_cast<const uint8_t*>(o.a), 2 * o.lda, 2 * o.ldga};
  const AnyOperand B{static_cast<const uint8_t*>(o.b), 2 * o.ldb, 0};
  const uint64_t tiles = product_tiles(MODE, P, NT, 128), cap = D.prof.sm_count;
  return launch_rows(kernel, (unsigned)(tiles < cap ? tiles : cap), kCopyThreads + 32 * (1 + kAnyOut), smem, D.stream, 1, A,
                     B, P, out);
}

template <int MODE, typename T>
int run(const DeviceSlot& D, const Operands& o, const ProductArgs& P, const StoreTile<MODE, T>& out) {
  if (tma_reads(MODE, P, o)) return launch_product_pair<MODE>(D, o, P, out);
  return launch_any<MODE, T, 128, 4>(D, o, P, out);
}

int check_site(const MapalProductSite* s) {
  if (!s) return set_error(MAPAL_ERR_INVALID, "site is null");
  if (s->dtype != MAPAL_DTYPE_F16 && s->dtype != MAPAL_DTYPE_BF16)
    return set_error(MAPAL_ERR_INVALID, "products are of f16 or bf16 rows");
  if ((s->ytype != s->dtype && s->ytype != MAPAL_DTYPE_F32) || (s->dwtype != s->dtype && s->dwtype != MAPAL_DTYPE_F32))
    return set_error(MAPAL_ERR_INVALID, "Y and dW are of the rows' type or f32");
  if (s->groups == 0 || s->groups > 65535) return set_error(MAPAL_ERR_INVALID, "1 to 65535 groups");
  // a tile's last row or column is counted in 32 bits
  const uint64_t most = 0x7fffff00ull;
  if (s->m > most || s->n > most || s->k > most) return set_error(MAPAL_ERR_UNSUPPORTED, "m, n or k over 2^31 - 256");
  return 0;
}

int check_rows(uint64_t rows, uint64_t cols, uint64_t ld, int dtype) {
  if (!rows_ok(rows, cols, ld, dtype_bytes(dtype)))
    return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
  return 0;
}

int check_matrices(const MapalProductSite& s, uint64_t ld, uint64_t ldg, int dtype) {
  MAPAL_TRY(check_rows(s.n, s.k, ld, dtype));
  const uint64_t one = s.n && s.k ? (s.n - 1) * ld + s.k : 0;
  if (s.groups > 1 && !rows_ok(s.groups, one, ldg, dtype_bytes(dtype)))
    return set_error(MAPAL_ERR_INVALID, "the stride between groups is shorter than a matrix, or too long");
  return 0;
}

bool on_type(const void* p, int dtype) { return ((uintptr_t)p & (dtype_bytes(dtype) - 1)) == 0; }

ProductArgs args_of(const DeviceSlot& D, const MapalProductSite& s, const int32_t* offsets) {
  ProductArgs P{};
  P.offsets = offsets;
  P.trap = D.trap;
  P.groups = s.groups;
  P.m = (uint32_t)s.m;
  P.parts = 1;
  P.bf16 = s.dtype == MAPAL_DTYPE_BF16;
  return P;
}

template <int MODE>
int by_type(const DeviceSlot& D, const Operands& o, const ProductArgs& P, int dtype, void* out, uint64_t ld, uint64_t ldg) {
  auto go = [&](auto t) {
    using T = decltype(t);
    return run<MODE, T>(D, o, P, StoreTile<MODE, T>{static_cast<T*>(out), ld, ldg});
  };
  if (dtype == MAPAL_DTYPE_F16) return go(__half{});
  if constexpr (MODE != kGradX)  // dX is of the rows' type
    if (dtype == MAPAL_DTYPE_F32) return go(float{});
  return go(__nv_bfloat16{});
}

}  // namespace

extern "C" int mapal_gpu_product(MapalGpuCtx* ctx, const MapalProductSite* site, const void* x, const void* w,
                                 const int32_t* offsets, void* y) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site));
    const MapalProductSite& s = *site;
    MAPAL_TRY(check_rows(s.m, s.k, s.ldx, s.dtype));
    MAPAL_TRY(check_matrices(s, s.ldw, s.ldg, s.dtype));
    MAPAL_TRY(check_rows(s.m, s.n, s.ldy, s.ytype));
    if (!offsets && s.groups != 1) return set_error(MAPAL_ERR_INVALID, "several groups need offsets");
    if (s.m == 0 || s.n == 0) return 0;
    if (!y || (s.k && (!x || !w))) return set_error(MAPAL_ERR_INVALID, "null x, w or y");
    if (!on_type(x, s.dtype) || !on_type(w, s.dtype) || !on_type(y, s.ytype) || ((uintptr_t)offsets & 3))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    ProductArgs P = args_of(D, s, offsets);
    P.lanes = (uint32_t)s.n;
    P.depth = (uint32_t)s.k;
    MAPAL_TRY(by_type<kForward>(D, {w, x, s.ldw, s.ldg, s.ldx, s.n, s.k, s.k}, P, s.ytype, y, s.ldy, 0));
    return finish(ctx, 0, true);
  });
}

extern "C" int mapal_gpu_product_grad(MapalGpuCtx* ctx, const MapalProductSite* site, const void* x, const void* w,
                                      const int32_t* offsets, const void* dy, void* dx, void* dw) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site));
    const MapalProductSite& s = *site;
    MAPAL_TRY(check_rows(s.m, s.n, s.lddy, s.dtype));
    if (dx) {
      MAPAL_TRY(check_matrices(s, s.ldw, s.ldg, s.dtype));
      MAPAL_TRY(check_rows(s.m, s.k, s.lddx, s.dtype));
    }
    if (dw) {
      MAPAL_TRY(check_rows(s.m, s.k, s.ldx, s.dtype));
      MAPAL_TRY(check_matrices(s, s.lddw, s.lddg, s.dwtype));
    }
    if (!offsets && s.groups != 1) return set_error(MAPAL_ERR_INVALID, "several groups need offsets");
    const bool do_x = dx && s.m && s.k, do_w = dw && s.n && s.k;
    if (!do_x && !do_w) return 0;
    if (s.m && s.n && (!dy || (do_x && !w) || (do_w && !x))) return set_error(MAPAL_ERR_INVALID, "null x, w or dy");
    if (!on_type(x, s.dtype) || !on_type(w, s.dtype) || !on_type(dy, s.dtype) || !on_type(dx, s.dtype) ||
        !on_type(dw, s.dwtype) || ((uintptr_t)offsets & 3))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    ProductArgs P = args_of(D, s, offsets);
    P.lanes = (uint32_t)s.k;
    if (do_x) {
      P.depth = (uint32_t)s.n;
      MAPAL_TRY(by_type<kGradX>(D, {w, dy, s.ldw, s.ldg, s.lddy, s.n, s.k, s.n}, P, s.dtype, dx, s.lddx, 0));
    }
    if (do_w) {
      P.depth = 0;
      P.cols = (uint32_t)s.n;
      MAPAL_TRY(by_type<kGradW>(D, {x, dy, s.ldx, 0, s.lddy, s.m, s.k, s.n}, P, s.dwtype, dw, s.lddw, s.lddg));
    }
    return finish(ctx, 0, true);
  });
}

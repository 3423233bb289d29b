// product.cu — products in 16-bit floats with one matrix or one per group of rows,
// and their gradients (mapal_gpu_product*). No counterpart in the reference.
#include "product.cuh"

namespace cg = cooperative_groups;

namespace {

// ---- operands that TMA cannot read ---------------------------------------------------------
//
// Bases or strides off 16 bytes: copying warps bring such an operand's block of t into
// the layout that TMA would have given it. Both layouts are lines of 128 bytes (a
// K-major line is a lane's or column's 64 steps of t, an MN-major one 64 lanes or
// columns at one step), so one loop serves all products. A thread has 16 bytes of
// every 32nd line: lines so far apart, and a line's next blocks, begin at the same
// place in an aligned word of 16 bytes, so its shift is the same for a whole tile. It
// loads the two aligned words that hold its bytes, a block ahead, and shifts them on
// the way to shared memory. What does not exist is zeros, steps behind a group's last
// among them.

struct CopyOperand {
  const uint8_t* base;
  uint64_t ld, ldg;  // bytes
};

constexpr int kCopyThreads = 256;

template <bool MN, int LINES>
struct Lines {
  static constexpr int kTurns = (LINES * 8 + kCopyThreads - 1) / kCopyThreads;
  const uint8_t* at;  // the aligned word of this thread's first line at the block's t
  uint64_t ld;
  uint32_t sh;
  int32_t lines;  // K-major: lines from this thread's first on; MN-major: steps of t from its first on
  int32_t width;  // elements from this thread's first on: K-major of t, MN-major of lanes or columns
  uint4 a[kTurns], b[kTurns];

  // first: the address of (first lane or column, first step of t).
  __device__ __forceinline__ void set(uint32_t thread, const uint8_t* first, uint64_t ld_, uint32_t extent, uint32_t depth) {
    const uint32_t c = thread & 7, line = thread >> 3;
    const uint8_t* p = first + line * ld_ + c * 16;
    sh = (uint32_t)(uintptr_t)p & 15;
    at = p - sh;
    ld = ld_;
    lines = (int32_t)(MN ? depth : extent) - (int32_t)line;
    width = (int32_t)(MN ? extent : depth) - (int32_t)(c * 8);
  }
  static __device__ __forceinline__ int line_of(int i) { return MN ? (i & 1) * 32 : i * 32; }
  static __device__ __forceinline__ int chunk_of(int i) { return MN ? i >> 1 : 0; }
  // Elements of turn i's 16 bytes that exist, 0 to 8.
  __device__ __forceinline__ int have(int i) const {
    return line_of(i) < lines ? max(0, min(8, width - chunk_of(i) * 64)) : 0;
  }
  __device__ __forceinline__ bool whole() const { return (MN ? lines > 32 : width >= 8) && (!MN || width >= (kTurns > 2 ? 72 : 8)); }

  // No aligned word is read without one of the elements in it.
  __device__ __forceinline__ void load() {
    const bool all = whole();
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const uint4* w = reinterpret_cast<const uint4*>(at + line_of(i) * ld + chunk_of(i) * 128);
      const int n = all ? (MN || line_of(i) < lines ? 8 : 0) : have(i);
      a[i] = n > 0 ? __ldg(w) : make_uint4(0, 0, 0, 0);
      b[i] = n > 0 && sh + 2 * n > 16 ? __ldg(w + 1) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void store(uint32_t thread, uint8_t* tile) const {
    const uint32_t c = thread & 7, line = thread >> 3;
    uint8_t* to = tile + line * 128 + ((c ^ (line & 7)) << 4);
    const bool all = whole();
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      uint4 v = straddle(a[i], b[i], sh);
      if (!all) {
        const int n = have(i);
        uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = n >= 2 * k + 2 ? q[k] : n == 2 * k + 1 ? q[k] & 0xffffu : 0u;
        v = make_uint4(q[0], q[1], q[2], q[3]);
      }
      *reinterpret_cast<uint4*>(to + i * (32 * 128)) = v;
    }
  }
  __device__ __forceinline__ void next() {
    if (MN) {
      at += kStepK * ld;
      lines -= kStepK;
    } else {
      at += 128;
      width -= kStepK;
    }
  }
};

// The address of lane or column `first` of an operand at step t.
template <bool MN>
__device__ __forceinline__ const uint8_t* operand_at(const CopyOperand& o, uint64_t group, uint64_t first, uint64_t t) {
  return o.base + group * o.ldg + (MN ? t * o.ld + 2 * first : first * o.ld + 2 * t);
}

// One CTA a tile of 128 lanes by NT columns, both operands copied.

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

template <int MODE, typename T, int NT, int STAGES>
__global__ void __launch_bounds__(kCopyThreads + 32 * (1 + kAnyOut), 1)
    product_any_kernel(const CopyOperand A, const CopyOperand B, const __grid_constant__ ProductArgs P,
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
  JobWalk<MODE, NT, 128> walk(P, blockIdx.x, gridDim.x);
  Job j;
  bool more = walk.now(j);
  uint32_t it = 0;

  if (warp < kCopy) {
    // ---- copies ----
    Lines<MODE != kForward, 128> la;
    Lines<MODE == kGradW, NT> lb;
    for (; more; more = walk.next(j)) {
      la.set(threadIdx.x, operand_at<MODE != kForward>(A, MODE == kGradW ? 0 : j.group, j.lane0, j.t0), A.ld,
             P.lanes - j.lane0, j.depth);
      lb.set(threadIdx.x, operand_at<MODE == kGradW>(B, 0, j.col0, j.t0), B.ld, j.cols, j.depth);
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
        la.store(threadIdx.x, sm.stage[s]);
        lb.store(threadIdx.x, sm.stage[s] + 128 * 128);
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
    for (; more; more = walk.next(j), ++n) {
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
    for (; more; more = walk.next(j), ++n) {
      const uint32_t b = n & 1;
      if (any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort)) {
        *abort = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      out.put_plain(P, j, tmem + ((uint32_t)(quarter * 32) << 16) + b * NT, j.lane0 + quarter * 32, 0, NT);
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

// ---- a CTA a tile ------------------------------------------------------------------------
//
// Products of few tiles: up to 128 columns (NT) and CH lanes. The MMA always has
// M = 128; with CH below 128 the other rows of its operand are whatever shared memory
// holds and their results are not read: few rows are bound by reading the weights, and
// narrower tiles spread them over more SMs.
//
// Where even that leaves SMs idle, t is split over a cluster of `split` CTAs: each
// leaves its f32 partial sums in the shared memory of the CTA that writes those
// columns, which adds them up in the CTAs' order.
//
// A stage holds KB blocks of t. Forward weights come with one load a stage where k
// and n allow it (multiples of 64 and 8): the map splits k into blocks and channels
// into eights, so that a stage lies as [eight][block][8 rows][128 bytes] and each row
// is read KB*128 bytes at a time. An MN-major operand comes as 64 lanes or columns by
// KB*64 steps with a load. grad w: rows behind a group's last are cleared as in pairs.

template <int NT, int CH, int KB, int STAGES>
struct TileSmem {
  static constexpr int kATile = CH * 128, kBTile = NT * 128;
  static constexpr int kStage = KB * (kATile + kBTile);
  // KB blocks of A, then of B; 1024-byte aligned for the swizzle. The MMA reads 128
  // lanes of A, in the last stage past its end.
  uint8_t stage[STAGES][kStage];
  uint8_t past[128 - CH > NT ? KB * (128 - CH - NT) * 128 : 16];
  uint64_t full[STAGES], empty[STAGES];
  uint64_t to_fix, fixed;  // a last block to clear has landed; it is cleared
  uint64_t acc_full[2], acc_empty[2];
  uint64_t parts, drained;
  alignas(16) uint8_t scratch[out_warps(NT)][kOutScratch];
  uint32_t tmem_base;
  int abort;
};

struct TileArgs {
  void* out;
  uint64_t ld, ldg;
  int32_t otype;
  uint32_t split;
  uint32_t wide;    // see StoreTile
  uint32_t folded;  // forward: A's map brings a whole stage at once
};

// f(typed pointer) for the output's type.
template <typename F>
__device__ __forceinline__ void with_type(const TileArgs& O, F&& f) {
  if (O.otype == MAPAL_DTYPE_BF16)
    f(static_cast<__nv_bfloat16*>(O.out));
  else if (O.otype == MAPAL_DTYPE_F16)
    f(static_cast<__half*>(O.out));
  else
    f(static_cast<float*>(O.out));
}

__host__ __device__ constexpr int tile_threads(int mode, int nt) { return 64 + 32 * out_warps(nt) + (mode == kGradW ? 32 : 0); }

template <int MODE, int NT, int CH, int KB, int STAGES>
__global__ void __launch_bounds__(tile_threads(MODE, NT), 1)
    product_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ ProductArgs P, const __grid_constant__ TileArgs O) {
  using Smem = TileSmem<NT, CH, KB, STAGES>;
  // two accumulators of NT columns; 16 of them are read with the 16 columns behind
  constexpr uint32_t kCols = NT < kTurnCols ? 2 * kTurnCols : 2 * NT;
  static_assert(NT + (NT < kTurnCols ? kTurnCols : NT) <= kCols, "the second accumulator's reads stay in what is allocated");
  constexpr int kOut = out_warps(NT);
  constexpr bool MN = MODE != kForward, MB = MODE == kGradW;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t split = O.split, rank = split > 1 ? blockIdx.x % split : 0;
  const uint64_t first = blockIdx.x / split, step = gridDim.x / split;
  volatile int* abort = &sm.abort;

  if (warp == 0 && elect_one()) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.to_fix, 1);
    mbar_init(&sm.fixed, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], kOut / 4 * (CH / 32));
    }
    mbar_init(&sm.parts, 1);
    mbar_init(&sm.drained, 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (split > 1 && warp == 0 && elect_one()) mbar_expect_tx(&sm.parts, NT * CH * 4);  // all CTAs' shares
  grid_wait();
  grid_go();
  JobWalk<MODE, NT, CH> walk(P, first, step);
  Job j;
  bool more = walk.now(j);
  uint32_t it = 0;  // stages taken, by the loads' and by the products' lane

  uint32_t fixes = 0;  // last blocks cleared
  uint32_t kb_lo, kbs, fills;  // this CTA's blocks of the tile, and the stages they take
  auto cut = [&]() {
    const uint32_t k_blocks = (j.depth + kStepK - 1) / kStepK;
    kb_lo = split > 1 ? (uint32_t)((uint64_t)k_blocks * rank / split) : 0;
    kbs = (split > 1 ? (uint32_t)((uint64_t)k_blocks * (rank + 1) / split) : k_blocks) - kb_lo;
    fills = (kbs + KB - 1) / KB;
  };
  if (more) cut();
  // whether the CTA's last block holds rows that are not the group's
  auto to_fix = [&]() {
    return MODE == kGradW && kbs && (j.depth & 15) && (kb_lo + kbs) * kStepK > j.depth && j.t0 + j.depth < P.m;
  };
  auto blocks_of = [&](uint32_t fill) { return min((uint32_t)KB, kbs - fill * KB); };
  const bool folded = !MN && KB > 1 && O.folded;
  auto load = [&](uint32_t fill) {
    const uint32_t s = it % STAGES, blocks = blocks_of(fill);
    uint8_t* st = sm.stage[s];
    const int t0 = (int)(j.t0 + (kb_lo + fill * KB) * kStepK);
    mbar_expect_tx(&sm.full[s], (MN || folded ? KB : blocks) * Smem::kATile + (MB ? KB : blocks) * Smem::kBTile);
    if (MN) {
#pragma unroll
      for (int c = 0; c < CH / 64; ++c) {
        uint8_t* to = st + c * (KB * kStepK * 128);
        if (MODE == kGradW)
          tma_load_2d(to, &map_a, (int)j.lane0 + c * 64, t0, &sm.full[s]);
        else
          tma_load_3d(to, &map_a, (int)j.lane0 + c * 64, t0, (int)j.group, &sm.full[s]);
      }
    } else if (folded) {
      tma_load_5d(st, &map_a, 0, 0, (int)(kb_lo + fill * KB), (int)(j.lane0 / 8), (int)j.group, &sm.full[s]);
    }
    if (MB) {
#pragma unroll
      for (int c = 0; c < NT / 64; ++c)
        tma_load_2d(st + KB * Smem::kATile + c * (KB * kStepK * 128), &map_b, (int)j.col0 + c * 64, t0, &sm.full[s]);
    }
#pragma unroll
    for (uint32_t u = 0; u < KB; ++u)
      if (u < blocks) {
        const int t = t0 + (int)u * kStepK;
        if (!MN && !folded) tma_load_3d(st + u * Smem::kATile, &map_a, t, (int)j.lane0, (int)j.group, &sm.full[s]);
        if (!MB) tma_load_2d(st + KB * Smem::kATile + u * Smem::kBTile, &map_b, t, (int)j.col0, &sm.full[s]);
      }
    ++it;
  };
  // the first stages are on their way before the others have begun
  if (warp == 0 && more && elect_one())
    while (it < STAGES && it < fills) load(it);
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(&sm.tmem_base)),
                 "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ---- loads ----
    uint32_t fill = it;  // of the first tile, some are issued
    for (; more; more = walk.next(j), fill = 0) {
      cut();
      if (elect_one())
        for (; fill < fills; ++fill) {
          if (!mbar_wait(&sm.empty[it % STAGES], ((it / STAGES) & 1) ^ 1, abort)) {
            *abort = 1;
            break;
          }
          load(fill);
        }
      if (any_of(*abort)) break;
    }
  } else if (warp == 1) {
    // ---- products ----
    uint32_t n = 0;
    for (; more; more = walk.next(j), ++n) {
      const uint32_t b = n & 1;
      cut();
      const bool fix = to_fix();
      if (elect_one()) {
        const uint32_t idesc = idesc_f16<MODE>(P.bf16, 128, (int)((j.cols + 15) / 16 * 16));
        if (!mbar_wait(&sm.acc_empty[b], ((n >> 1) & 1) ^ 1, abort)) *abort = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (uint32_t fill = 0; fill < fills && !*abort; ++fill, ++it) {
          const uint32_t s = it % STAGES, blocks = blocks_of(fill);
          bool ok = mbar_wait(&sm.full[s], (it / STAGES) & 1, abort);
          if (fix && fill + 1 == fills && ok) {
            // the clearing warp is told here: a wait of its own on the stage would have to follow every one of its uses
            mbar_arrive(&sm.to_fix);
            ok = mbar_wait(&sm.fixed, fixes++ & 1, abort);
          }
          if (!ok) {
            *abort = 1;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = MN ? desc_mn(sm.stage[s], KB * kStepK * 128) : desc128(sm.stage[s], folded ? KB * 1024 : 1024),
                         db = MB ? desc_mn(sm.stage[s] + KB * Smem::kATile, KB * kStepK * 128)
                                 : desc128(sm.stage[s] + KB * Smem::kATile);
          const uint32_t next = (MN ? kStepK * 128 : folded ? 1024 : Smem::kATile) >> 4;
          const uint32_t next_b = (MB ? kStepK * 128 : Smem::kBTile) >> 4;
#pragma unroll
          for (uint32_t u = 0; u < KB; ++u)
            if (u < blocks) {
              // grad w: no step behind the group's rows
              const uint32_t left = j.depth - (kb_lo + fill * KB + u) * kStepK;
#pragma unroll
              for (uint32_t kk = 0; kk < kStepK / 16; ++kk)
                if (MODE != kGradW || kk * 16 < left)
                  mma_f16<1>(tmem + b * NT, da + u * next + kk * operand_step<MN>(), db + u * next_b + kk * operand_step<MB>(),
                             idesc, fill > 0 || u > 0 || kk > 0);
            }
          mma_commit(&sm.empty[s]);
        }
        mma_commit(&sm.acc_full[b]);
      }
      if (any_of(*abort)) break;
    }
  } else if (MODE == kGradW && warp == 2 + kOut) {
    // ---- last blocks: rows behind the group's become zeros ----
    for (; more; more = walk.next(j)) {
      cut();
      it += fills;
      if (!to_fix()) continue;
      const uint32_t s = (it - 1) % STAGES;
      if (any_of(!mbar_wait(&sm.to_fix, fixes++ & 1, abort))) {
        *abort = 1;
        break;
      }
      const uint32_t rows = j.depth - (kb_lo + (fills - 1) * KB) * kStepK, to = (rows + 15) / 16 * 16;
      for (uint32_t chunk = 0; chunk < (CH + NT) / 64; ++chunk)
        for (uint32_t i = rows * 8 + lane; i < to * 8; i += 32)
          *reinterpret_cast<uint4*>(sm.stage[s] + chunk * (KB * kStepK * 128) + i * 16) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.fixed);
    }
  } else if ((warp & 3) < CH / 32) {
    // ---- output ----
    const int quarter = warp & 3;  // TMEM lanes 32*quarter to +31
    uint32_t n = 0;
    for (; more; more = walk.next(j), ++n) {
      cut();
      const uint32_t b = n & 1;
      const uint32_t from = (warp - 2) / 4 * (NT / (kOut / 4));
      if (any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort)) {  // *abort: its commit was an aborted tile's
        *abort = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (split > 1) break;  // a cluster's one tile is joined below
      with_type(O, [&](auto* out) {
        StoreTile<MODE, std::remove_pointer_t<decltype(out)>>{out, O.ld, O.ldg, O.wide != 0}.put(
            P, j, tmem + ((uint32_t)(quarter * 32) << 16) + b * NT, j.lane0 + quarter * 32, from, from + NT / (kOut / 4),
            sm.scratch[warp - 2]);
      });
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
    }
  }

  if (split > 1) {
    // ---- the cluster's tile: its parts of t joined ----
    // Every CTA's products are done, so its stages are free: the partial sums go there, [column][lane], and on to the
    // CTAs that write them as one bulk copy each. (Stores to other CTAs lane by lane took 8 us for 128 x 128.)
    __syncwarp();
    cg::this_cluster().sync();
    if (more && warp >= 2 && warp < 2 + kOut && (warp & 3) < CH / 32 && !any_of(*abort)) {
      constexpr int kPart = NT * CH * 4;
      static_assert(2 * kPart <= (int)sizeof(sm.stage), "own and received sums");
      const uint32_t quarter = warp & 3, share = NT / split, half = (warp - 2) / 4;
      float* mine = reinterpret_cast<float*>(sm.stage[0]) + quarter * 32 + lane;
      const float* received = mine + NT * CH;
      for (uint32_t k0 = half * (NT / (kOut / 4)); k0 < (half + 1) * (NT / (kOut / 4)); k0 += 16) {
        float f[16];
        tmem_ld16f(tmem + ((quarter * 32) << 16) + k0, f);
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[(k0 + i) * CH] = kbs ? f[i] : 0.0f;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("bar.sync 1, %0;" ::"n"(kOut / 4 * CH) : "memory");  // the writing warps
      if (warp == (CH == 128 ? 2 : 4) && elect_one())                  // the first of them
        for (uint32_t q = 0; q < split; ++q)
          asm volatile(
              "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                  remote(sa(sm.stage[0]) + kPart + rank * share * CH * 4, q)),
              "r"(sa(sm.stage[0]) + q * share * CH * 4), "r"(share * CH * 4), "r"(remote(sa(&sm.parts), q))
              : "memory");
      if (any_of(!mbar_wait_cluster(&sm.parts, 0, abort))) {
        *abort = 1;
      } else {
        const uint32_t own = share / (kOut / 4), i0 = half * own, j0 = rank * share + i0, at = j.lane0 + quarter * 32 + lane;
        with_type(O, [&](auto* out) {
          using T = std::remove_pointer_t<decltype(out)>;
          T* c = out + (MODE == kGradW ? (uint64_t)j.group * O.ldg : 0) + (uint64_t)(j.col0 + j0) * O.ld + at;
          constexpr uint32_t kTurn = NT / 8 / (kOut / 4) < 8 ? NT / 8 / (kOut / 4) : 8;  // columns at once; split is at most 8
          for (uint32_t i = 0; i < own && j0 + i < j.cols; i += kTurn, c += kTurn * O.ld) {
            float acc[kTurn] = {};
#pragma unroll 2
            for (uint32_t q = 0; q < split; ++q)
#pragma unroll
              for (uint32_t u = 0; u < kTurn; ++u) acc[u] += received[(q * share + i0 + i + u) * CH];
#pragma unroll
            for (uint32_t u = 0; u < kTurn; ++u)
              if (at < P.lanes && j0 + i + u < j.cols) c[u * O.ld] = from_f32<T>(acc[u]);
          }
        });
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (split > 1)
    cg::this_cluster().sync();  // nobody leaves while another may still write here
  else
    __syncthreads();
  if (*abort) {
    // a wait gave up: what is still in flight ends before shared memory and TMEM are given back
    if (warp == 0 && elect_one()) {
      atomicOr(P.trap, kDeviceTimeout);
      for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i)
        mbar_wait(&sm.full[i % STAGES], (i / STAGES) & 1, nullptr);
    }
    if (warp == 1 && elect_one()) {
      mma_commit(&sm.drained);
      mbar_wait(&sm.drained, 0, nullptr);
    }
    __syncthreads();
  }
  if (warp == 1) {
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
  const CopyOperand A{static_cast<const uint8_t*>(o.a), 2 * o.lda, 2 * o.ldga};
  const CopyOperand B{static_cast<const uint8_t*>(o.b), 2 * o.ldb, 0};
  const uint64_t tiles = product_tiles(MODE, P, NT, 128), cap = D.prof.sm_count;
  return launch_rows(kernel, (unsigned)(tiles < cap ? tiles : cap), kCopyThreads + 32 * (1 + kAnyOut), smem, D.stream, 1, A,
                     B, P, out);
}

// A way to cut the product: lanes and columns of a tile, parts of t; pairs of CTAs
// have 256 lanes.
struct Cut {
  uint32_t lanes, cols, split;
};

// Cycles of a cut, from what bounds its tiles: the MMA (N/2 cycles for 128 lanes and
// 16 steps of t, 72 + N/4 at least), and the loads, at up to 58 bytes a cycle for
// an SM and 7200 for all; tiles run in waves. The constants are fitted to 210 products
// (1 to 16000 rows, 64 to 8192 channels, 1 to 64 matrices, all three modes) that were
// measured with every cut. grad w: a group's rows are on the device, and the mean
// stands for each, which groups of very different sizes are cut the worse for.
double cycles_of(int mode, const ProductArgs& P, const Cut& c, uint32_t depth, int sms) {
  const bool pair = c.lanes == 256;
  const double tiles = (double)product_tiles(mode, P, c.cols, c.lanes) * c.split, at_once = pair ? sms / 2 : sms;
  const double active = tiles < at_once ? tiles : at_once, ctas = pair ? 2 * active : active;
  const double blocks = (double)((depth + kStepK - 1) / kStepK) / c.split;
  const double rate = 7200.0 / ctas < 58.0 ? 7200.0 / ctas : 58.0;
  const double load = (pair ? 256 : c.lanes + c.cols) * 128.0 / rate;
  const uint32_t have = mode == kGradW ? P.cols : P.m;
  const double cols = have < c.cols ? (double)((have + 15) / 16 * 16) : c.cols;
  const double mma = 4 * (cols / 4 + 72 > cols / 2 ? cols / 4 + 72 : cols / 2);
  const double size = c.lanes * c.cols / 16384.0, waves = (double)(uint64_t)((tiles + at_once - 1) / at_once);
  return (pair ? 9900 : 5200) + waves * (blocks * (load > mma ? load : mma) + (pair ? 2000 : 860 * size) + 1500) +
         (c.split > 1 ? 3300 + 3500 * size : 0);
}

// W as [group][eight channels][block of k][8][64], in boxes of lanes/8 x blocks.
int folded_map(CUtensorMap* map, const ProductArgs& P, const Operands& o, uint32_t lanes, uint32_t blocks) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dim[5] = {(cuuint64_t)kStepK, 8, o.a_cols / kStepK, o.rows / 8, P.groups};
  cuuint64_t stride[4] = {2 * o.lda, 128, 16 * o.lda, 2 * (P.groups > 1 ? o.ldga : o.rows * o.lda)};
  cuuint32_t box[5] = {(cuuint32_t)kStepK, 8, blocks, lanes / 8, 1}, one[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, const_cast<void*>(o.a), dim, stride, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return 0;
}

template <int MODE, int NT, int CH, int KB, int STAGES>
int launch_tile(const DeviceSlot& D, const Operands& o, const ProductArgs& P, TileArgs O) {
  using Smem = TileSmem<NT, CH, KB, STAGES>;
  CUtensorMap ma, mb;
  O.folded = MODE == kForward && KB > 1 && o.a_cols % kStepK == 0 && o.rows % 8 == 0 && o.lda < (1ull << 35);
  const uint64_t mats = MODE == kGradW ? 1 : P.groups;
  if (O.folded)
    MAPAL_TRY(folded_map(&ma, P, o, CH, KB));
  else
    MAPAL_TRY(product_map(&ma, o.a, o.rows, o.a_cols, o.lda, mats, o.ldga, MODE == kGradW ? 2 : 3,
                          MODE == kForward ? CH : KB * kStepK));
  MAPAL_TRY(product_map(&mb, o.b, P.m, o.b_cols, o.ldb, 1, 0, 2, MODE == kGradW ? KB * kStepK : NT));
  constexpr size_t most = sizeof(Smem) + 1024;
  static_assert(most <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  auto kernel = product_tile_kernel<MODE, NT, CH, KB, STAGES>;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, most, "product shared memory"));
  const uint64_t tiles = product_tiles(MODE, P, NT, CH), cap = O.split > 1 ? tiles : (uint64_t)D.prof.sm_count;
  return launch_rows(kernel, (unsigned)((tiles < cap ? tiles : cap) * O.split), tile_threads(MODE, NT),
                     most, D.stream, O.split, ma, mb, P, O);
}

template <int MODE, typename T>
int run(const DeviceSlot& D, const Operands& o, const ProductArgs& P, const StoreTile<MODE, T>& out, int otype) {
  const bool ta = tma_reads_a(MODE, P, o), tb = tma_reads_b(P, o);
  if (!ta || !tb) {
    const bool ra = raw_reads(o.rows, o.a_cols, o.lda, MODE == kGradW ? 1 : P.groups, o.ldga);
    if (!ra || !raw_reads(P.m, o.b_cols, o.ldb, 1, 0)) return launch_any<MODE, T, 128, 4>(D, o, P, out);
    if (ta) return launch_product_pair<MODE, false, true>(D, o, P, out);
    if (tb) return launch_product_pair<MODE, true, false>(D, o, P, out);
    return launch_product_pair<MODE, true, true>(D, o, P, out);
  }
  static constexpr Cut kCuts[] = {{256, 256, 1}, {128, 128, 1}, {64, 128, 1}, {128, 64, 1}, {64, 64, 1},
                                  {128, 32, 1},  {64, 32, 1},   {128, 16, 1}, {64, 16, 1},  {32, 16, 1}};
  // grad w: the groups' rows are on the device; the mean stands for each
  const uint32_t depth = MODE == kGradW ? (P.m + P.groups - 1) / P.groups : P.depth, blocks = (depth + kStepK - 1) / kStepK;
  Cut best{};
  double least = 0;
  for (Cut c : kCuts) {
    if (MODE == kGradX && c.lanes == 32) continue;                        // an MN-major line is 64 lanes,
    if (MODE == kGradW && (c.cols < 128 || c.lanes < 128)) continue;      // or columns
    for (c.split = 1; c.split <= 8; c.split *= 2) {
      if (c.split > 1 && (c.lanes == 256 || (c.cols == 128 && c.lanes == 64) || c.split * 4 > blocks ||
                          product_tiles(MODE, P, c.cols, c.lanes) * c.split > (uint64_t)D.prof.sm_count))
        break;
      const double cy = cycles_of(MODE, P, c, depth, D.prof.sm_count);
      if (best.lanes == 0 || cy < least) {
        best = c;
        least = cy;
      }
    }
  }
  const TileArgs O{out.out, out.ld, out.ldg, otype, best.split, out.wide, 0};
  switch (best.lanes * 1000 + best.cols) {
    case 256256: return launch_product_pair<MODE, false, false>(D, o, P, out);
    case 128128:
      return launch_tile<MODE, 128, 128, 2, 3>(D, o, P, O);
  }
  if constexpr (MODE != kGradW) {
    switch (best.lanes * 1000 + best.cols) {
      case 64128: return launch_tile<MODE, 128, 64, 2, 4>(D, o, P, O);
      case 128064: return launch_tile<MODE, 64, 128, 2, 3>(D, o, P, O);
      case 64064: return launch_tile<MODE, 64, 64, 2, 6>(D, o, P, O);
      case 128032: return launch_tile<MODE, 32, 128, 2, 5>(D, o, P, O);
      case 64032: return launch_tile<MODE, 32, 64, 4, 4>(D, o, P, O);
      case 128016: return launch_tile<MODE, 16, 128, 2, 5>(D, o, P, O);
      case 64016: return launch_tile<MODE, 16, 64, 4, 4>(D, o, P, O);
    }
    if constexpr (MODE == kForward) return launch_tile<MODE, 16, 32, 4, 7>(D, o, P, O);
  }
  return set_error(MAPAL_ERR_UNSUPPORTED, "no tile for this product");
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
    const uint64_t rows = MODE == kGradW ? P.cols : P.m;
    const bool wide = aligned16(out) && (rows == 1 || ld % 8 == 0) && (MODE != kGradW || P.groups == 1 || ldg % 8 == 0);
    return run<MODE, T>(D, o, P, StoreTile<MODE, T>{static_cast<T*>(out), ld, ldg, wide}, dtype);
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
    if (s.k && (y == x || y == w)) return set_error(MAPAL_ERR_INVALID, "y is x or w");
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
    // an output may be an operand that the call does not read: x without dw, w without dx
    const bool reads = s.m && s.n;
    if (reads && ((do_x && (dx == dy || dx == w || (do_w && dx == x))) || (do_w && (dw == dy || dw == x || (do_x && dw == w)))))
      return set_error(MAPAL_ERR_INVALID, "dx or dw is an array that the call reads");
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

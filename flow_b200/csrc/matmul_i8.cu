// matmul_i8.cu — products in 8-bit integers with a scale for each row of A and
// each row (output channel) of B, for one matrix or one per group of rows
// (mapal_gpu_matmul_i8). No counterpart in the reference.
//
// C[i, j] = (sum_k A[i, k]*B[g][j, k]) * scale_a[i] * scale_b[g][j]. The sum
// is exact in 32 bits for k < 2^17 (127^2 and even 128^2 times k stays below
// 2^31), so any split or order of it gives the same bits; the float steps are
// one conversion and two multiplications, each rounded to f32.
#include <cooperative_groups.h>

#include "f32x2.cuh"
#include "rows.cuh"
#include "tcgen05.cuh"
#include "tiles.cuh"

namespace cg = cooperative_groups;

namespace {

template <typename T>
__device__ __forceinline__ T scaled(int acc, float sa, float sb) {
  return from_f32<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc), sa), sb));
}

// ---- tensor cores ------------------------------------------------------------------
//
// The product is taken as D = B*A^T: B's rows (channels) are the M dimension
// of tcgen05.mma and A's rows (tokens) the N dimension, so that a tile may be
// as narrow in tokens as there are tokens (16 at least) while the weights,
// which a small batch spends its time reading, always fill the lanes, and so
// that neighbouring lanes hold neighbouring elements of a row of C.
//
// Both kernels have the same roles:
//   warp 0     walks the tiles; one lane issues the TMA loads of each 128-byte
//              block of k (128-byte swizzle) into a ring of STAGES stages. k's
//              tail and channels beyond n read as zeros;
//   warp 1     allocates TMEM (two accumulators, so the next tile's products
//              run beside this tile's output) and issues kind::i8, K32, with N
//              the tile's tokens rounded up;
//   the others read the accumulator, scale and store C.
// TMEM is taken after grid_wait: no kernel holds it while it waits for the one
// before it, which may still have to take its own. A wait that gave up ends its
// whole warp together (any_of), since every step of a tile is a warp's.
// Tiles are numbered channel tiles first, then token tiles, then groups, and a
// persistent grid takes every gridDim-th; each warp finds a tile's group by a
// scan over the offsets, 32 groups at a time.

// D 32-bit integers, A and B signed 8-bit, both K-major.
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <int CTAS>
__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

struct TcArgs {
  const int32_t* offsets;
  const float* sa;
  const float* sb;
  void* C;
  unsigned* trap;
  uint64_t ldc;
  uint32_t m, n, k_blocks, groups, split;
  uint32_t folded;  // the weights' map brings a whole stage at once (single CTAs)
};

// The scales of tokens [from, to), into shared memory of the warp's own, before
// the accumulator is ready: a load for each token in put_tile would wait its
// turn behind the stores before it, 90 ns a token.
__device__ __forceinline__ void take_scales(const TcArgs& P, const Tile& t, uint32_t from, uint32_t to, float* scales) {
  to = min(to, t.tokens);
  __syncwarp();
  for (uint32_t j = from + (threadIdx.x & 31); j < to; j += 32)
    scales[j - from] = P.sa ? __ldg(P.sa + t.token0 + j) : 1.0f;
  __syncwarp();
}

// Tokens [from, to) of a warp's 32 lanes of the accumulator, 16 at a time, to C.
// A warp is alone with its latencies here, so the instructions a token are kept
// few: products on pairs of tokens, one conversion for two.
template <typename T>
__device__ __forceinline__ void put_tile(const TcArgs& P, const Tile& t, uint32_t taddr, uint32_t channel, float sb,
                                         uint32_t from, uint32_t to, const float* scales) {
  const bool in = channel < P.n;
  to = min(to, t.tokens);
  T* c = static_cast<T*>(P.C) + (uint64_t)(t.token0 + from) * P.ldc + (in ? channel : 0);
  const f2 sb2 = f2_splat(sb);
  for (uint32_t j0 = from; j0 < to; j0 += 16, scales += 16) {
    int r[16];
    tmem_ld16(taddr + j0, r);
    if (j0 + 16 <= to && in) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 s = *reinterpret_cast<const float4*>(scales + j);
        const f2 v0 = f2_mul(f2_mul(f2_pack(__int2float_rn(r[j]), __int2float_rn(r[j + 1])), f2_pack(s.x, s.y)), sb2);
        const f2 v1 = f2_mul(f2_mul(f2_pack(__int2float_rn(r[j + 2]), __int2float_rn(r[j + 3])), f2_pack(s.z, s.w)), sb2);
        const float v[4] = {f2_lo(v0), f2_hi(v0), f2_lo(v1), f2_hi(v1)};
        Pack<T, 4> o;
        o.set(v);
        T w[4];
        memcpy(w, o.w, sizeof(w));
        c[0] = w[0];
        c[P.ldc] = w[1];
        c[2 * P.ldc] = w[2];
        c[3 * P.ldc] = w[3];
        c += 4 * P.ldc;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j, c += P.ldc)
        if (in && j0 + j < to) *c = scaled<T>(r[j], scales[j], sb);
    }
  }
}

// ---- one CTA a tile ----------------------------------------------------------------
//
// Up to 128 tokens (NT) and CH channels. The MMA always has M = 128; with CH
// below 128 the other rows of its operand are whatever shared memory holds and
// their results are not read: a small batch is bound by reading the weights,
// and narrower tiles spread them over more SMs.
//
// Where even that leaves SMs idle, k is split over a cluster of `split` CTAs:
// each leaves its integer partial sums in the shared memory of the CTA that
// writes those tokens, which adds them up. Integer sums are exact in any order,
// so the split does not change a bit.

// Weights come with one load a stage where k and n allow it (multiples of 128
// and 8): the map splits k into blocks and channels into eights, so that a
// stage lies as [eight][block][8 rows][128 bytes] and each row is read 512
// bytes at a time, which HBM likes better than four visits of 128 (128 CTAs
// streaming 64 rows of 4096 bytes each: 6.6 against 7.9 us).
//
// A stage holds KB blocks of k, so that one wait, one commit and one round of
// the rings' bookkeeping (about 300 cycles in the loading lane, 140 of them a
// wait that succeeds at once) serve KB*4 MMAs of 64 cycles each.
template <int NT, int CH, int KB, int STAGES>
struct TcSmem {
  static constexpr int kWTile = CH * kBlockK, kXTile = NT * kBlockK;
  static constexpr int kStage = KB * (kWTile + kXTile);
  // KB blocks of weights, then of tokens; 1024-byte aligned for the swizzle.
  // The MMA reads 128 rows of weights, in the last stage past its end.
  uint8_t stage[STAGES][kStage];
  uint8_t past[128 - CH > NT ? KB * (128 - CH - NT) * kBlockK : 16];
  uint64_t full[STAGES], empty[STAGES];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t parts, drained;
  alignas(16) float scales[out_warps(NT)][kHalfTokens];
  uint32_t tmem_base;
  int abort;
};

template <typename T, int NT, int CH, int KB, int STAGES>
__global__ void __launch_bounds__(64 + 32 * out_warps(NT), 1)
    mm_i8_tc_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ TcArgs P) {
  using Smem = TcSmem<NT, CH, KB, STAGES>;
  constexpr uint32_t kCols = 2 * NT < 32 ? 32 : 2 * NT;
  constexpr int kOut = out_warps(NT);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  int* partial = reinterpret_cast<int*>(&sm + 1);  // split > 1: NT x CH partial sums
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t split = P.split, rank = split > 1 ? blockIdx.x % split : 0;
  const uint64_t first = blockIdx.x / split, step = gridDim.x / split;
  const uint32_t kb_lo = (uint32_t)((uint64_t)P.k_blocks * rank / split);
  const uint32_t kbs = (uint32_t)((uint64_t)P.k_blocks * (rank + 1) / split) - kb_lo;
  volatile int* abort = &sm.abort;

  if (warp == 0 && elect_one()) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], kOut / 4 * (CH / 32));
    }
    mbar_init(&sm.parts, split * CH);
    mbar_init(&sm.drained, 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  grid_wait();
  grid_go();
  TileWalk walk{P.offsets, P.groups, P.m, NT, CH, (P.n + CH - 1) / CH, P.trap};
  walk.load();
  Tile t;
  bool more = walk.at(first, t);
  uint32_t it = 0;  // stages taken, by the loads' and by the products' lane

  const uint32_t fills = (kbs + KB - 1) / KB;  // stages a tile takes
  auto blocks_of = [&](uint32_t fill) { return min((uint32_t)KB, kbs - fill * KB); };
  auto load = [&](uint32_t fill) {
    const uint32_t s = it % STAGES, blocks = blocks_of(fill);
    uint8_t* st = sm.stage[s];
    const bool folded = KB > 1 && P.folded;
    mbar_expect_tx(&sm.full[s], (folded ? KB : blocks) * Smem::kWTile + blocks * Smem::kXTile);
    if (folded)
      tma_load_5d(st, &map_w, 0, 0, (int)(kb_lo + fill * KB), (int)(t.channel0 / 8), (int)t.group, &sm.full[s]);
#pragma unroll
    for (uint32_t u = 0; u < KB; ++u)
      if (u < blocks) {
        const int k0 = (int)(kb_lo + fill * KB + u) * kBlockK;
        if (!folded) tma_load_3d(st + u * Smem::kWTile, &map_w, k0, (int)t.channel0, (int)t.group, &sm.full[s]);
        tma_load_2d(st + KB * Smem::kWTile + u * Smem::kXTile, &map_x, k0, (int)t.token0, &sm.full[s]);
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
  if (split > 1)
    cg::this_cluster().sync();  // the others' barriers are there before any arrival
  else
    __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ---- loads ----
    uint32_t fill = it;  // of the first tile, some are issued
    for (uint64_t tile = first; more; tile += step, more = walk.at(tile, t), fill = 0) {
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
    for (uint64_t tile = first; more; tile += step, more = walk.at(tile, t), ++n) {
      const uint32_t b = n & 1;
      if (elect_one()) {
        const uint32_t idesc = idesc_i8(128, (int)((t.tokens + 15) / 16 * 16));
        if (!mbar_wait(&sm.acc_empty[b], ((n >> 1) & 1) ^ 1, abort)) *abort = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (uint32_t fill = 0; fill < fills && !*abort; ++fill, ++it) {
          const uint32_t s = it % STAGES, blocks = blocks_of(fill);
          if (!mbar_wait(&sm.full[s], (it / STAGES) & 1, abort)) {
            *abort = 1;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dw = desc128(sm.stage[s], P.folded ? KB * 1024 : 1024),
                         dx = desc128(sm.stage[s] + KB * Smem::kWTile);
          const uint32_t next = P.folded ? 1024 >> 4 : Smem::kWTile >> 4;
#pragma unroll
          for (uint32_t u = 0; u < KB; ++u)
            if (u < blocks) {
#pragma unroll
              for (uint32_t kk = 0; kk < kBlockK / 32; ++kk)
                mma_i8<1>(tmem + b * NT, dw + u * next + kk * 2, dx + u * (Smem::kXTile >> 4) + kk * 2, idesc,
                          fill > 0 || u > 0 || kk > 0);
            }
          mma_commit(&sm.empty[s]);
        }
        mma_commit(&sm.acc_full[b]);
      }
      if (any_of(*abort)) break;
    }
  } else if ((warp & 3) < CH / 32) {
    // ---- scales and output ----
    const int quarter = warp & 3;  // TMEM lanes 32*quarter to +31
    uint32_t n = 0;
    for (uint64_t tile = first; more; tile += step, more = walk.at(tile, t), ++n) {
      const uint32_t b = n & 1;
      const uint32_t channel = t.channel0 + quarter * 32 + lane;
      const float sb = P.sb && channel < P.n ? __ldg(P.sb + (uint64_t)t.group * P.n + channel) : 1.0f;
      const uint32_t from = (warp - 2) / 4 * (NT / (kOut / 4));
      float* scales = sm.scales[warp - 2];
      if (split == 1) take_scales(P, t, from, from + NT / (kOut / 4), scales);
      if (any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort)) {  // *abort: its commit was an aborted tile's
        *abort = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t col = tmem + ((uint32_t)(quarter * 32) << 16) + b * NT;
      if (split == 1) {
        put_tile<T>(P, t, col, channel, sb, from, from + NT / (kOut / 4), scales);
      } else {
        const uint32_t share = NT / split;
        for (uint32_t k0 = 0; k0 < t.tokens; k0 += 16) {
          int r[16];
          tmem_ld16(col + k0, r);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t at = ((rank * share + (k0 + j) % share) * CH + quarter * 32 + lane) * 4;
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(remote(sa(partial) + at, (k0 + j) / share)), "r"(r[j])
                         : "memory");
          }
        }
        for (uint32_t q = 0; q < split; ++q) arrive_remote(remote(sa(&sm.parts), q));
        if (any_of(!mbar_wait_cluster(&sm.parts, 0, abort))) {
          *abort = 1;
          break;
        }
        // at most 32 tokens a CTA: split is 2 or more and NT at most 64
        const uint32_t j0 = rank * share;
        const float sv = P.sa && lane < share && j0 + lane < t.tokens ? __ldg(P.sa + t.token0 + j0 + lane) : 1.0f;
        T* c = static_cast<T*>(P.C) + (uint64_t)(t.token0 + j0) * P.ldc + channel;
        for (uint32_t j = 0; j < share && j0 + j < t.tokens; ++j, c += P.ldc) {
          int acc = 0;
          for (uint32_t q = 0; q < split; ++q) acc += partial[(q * share + j) * CH + quarter * 32 + lane];
          const float s = __shfl_sync(0xffffffffu, sv, j);
          if (channel < P.n) *c = scaled<T>(acc, s, sb);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
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

// ---- a pair of CTAs a tile ---------------------------------------------------------
//
// 256 channels and up to 256 tokens: each CTA of the pair loads its 128 channels
// and half of the tokens, and the pair's MMA (cta_group::2, issued by the first
// CTA) reads both halves from both, so a CTA moves 32 KB a block of k where a
// 128 x 256 tile of its own moves 48. Large products of single CTAs are bound by
// that traffic from L2 (about 11.6 TB/s): 8192^3 0.54 ms, where pairs take 0.39
// and are bound by the tensor pipe (84% of its cycles, measured on 2048 x 8192 x
// 8192) and, back to back, by the power limit (0.43 ms).

constexpr int kPairStages = 3, kPairKB = 2;
struct PairSmem {
  static constexpr int kHalf = 128 * kBlockK;  // of channels, and of tokens
  uint8_t stage[kPairStages][kPairKB * 2 * kHalf];
  uint64_t full[kPairStages];   // the first CTA's: both CTAs' loads have landed
  uint64_t empty[kPairStages];  // each CTA's own
  uint64_t acc_full[2];         // each CTA's own
  uint64_t acc_empty[2];        // the first CTA's: both CTAs have read the accumulator
  uint64_t drained;
  alignas(16) float scales[out_warps(256)][kHalfTokens];
  uint32_t tmem_base;
  int abort;
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + 32 * out_warps(256), 1)
    mm_i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                      const __grid_constant__ TcArgs P) {
  constexpr int NT = 256;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  PairSmem& sm = *reinterpret_cast<PairSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t rank = blockIdx.x & 1;
  const uint64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
  volatile int* abort = &sm.abort;

  if (warp == 0 && elect_one()) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 2 * out_warps(256));
    }
    mbar_init(&sm.drained, 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  grid_wait();
  grid_go();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(&sm.tmem_base)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cg::this_cluster().sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;
  TileWalk walk{P.offsets, P.groups, P.m, NT, 256, (P.n + 255) / 256, P.trap};
  walk.load();
  Tile t;
  bool more = walk.at(first, t);
  uint32_t it = 0;


  if (warp == 0) {
    // ---- loads, each CTA its halves, both counted by the first CTA's barrier ----
    for (uint64_t tile = first; more; tile += step, more = walk.at(tile, t)) {
      const int half = (int)((t.tokens + 31) / 32 * 16);  // tokens of each CTA
      if (elect_one())
        for (uint32_t kb = 0; kb < P.k_blocks; kb += kPairKB, ++it) {
          const uint32_t s = it % kPairStages, blocks = min((uint32_t)kPairKB, P.k_blocks - kb);
          if (!mbar_wait(&sm.empty[s], ((it / kPairStages) & 1) ^ 1, abort)) {
            *abort = 1;
            break;
          }
          if (rank == 0) mbar_expect_tx(&sm.full[s], blocks * 4 * PairSmem::kHalf);
          const uint32_t bar = remote(sa(&sm.full[s]), 0);
#pragma unroll
          for (uint32_t u = 0; u < kPairKB; ++u)
            if (u < blocks) {
              const int k0 = (int)(kb + u) * kBlockK;
              asm volatile(
                  "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
                  "{%2, %3, %4}], [%5];" ::"r"(sa(sm.stage[s] + 2 * u * PairSmem::kHalf)),
                  "l"(&map_w), "r"(k0), "r"((int)(t.channel0 + rank * 128)), "r"((int)t.group), "r"(bar)
                  : "memory");
              asm volatile(
                  "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
                  "{%2, %3}], [%4];" ::"r"(sa(sm.stage[s] + (2 * u + 1) * PairSmem::kHalf)),
                  "l"(&map_x), "r"(k0), "r"((int)t.token0 + (int)rank * half), "r"(bar)
                  : "memory");
            }
        }
      if (any_of(*abort)) break;
    }
  } else if (warp == 1) {
    // ---- products, by the first CTA ----
    uint32_t n = 0;
    for (uint64_t tile = first; rank == 0 && more; tile += step, more = walk.at(tile, t), ++n) {
      const uint32_t b = n & 1;
      if (elect_one()) {
        const uint32_t idesc = idesc_i8(256, (int)((t.tokens + 31) / 32 * 32));
        if (!mbar_wait_cluster(&sm.acc_empty[b], ((n >> 1) & 1) ^ 1, abort)) *abort = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (uint32_t kb = 0; kb < P.k_blocks && !*abort; kb += kPairKB, ++it) {
          const uint32_t s = it % kPairStages, blocks = min((uint32_t)kPairKB, P.k_blocks - kb);
          if (!mbar_wait(&sm.full[s], (it / kPairStages) & 1, abort)) {
            *abort = 1;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dw = desc128(sm.stage[s]), dx = desc128(sm.stage[s] + PairSmem::kHalf);
#pragma unroll
          for (uint32_t u = 0; u < kPairKB; ++u)
            if (u < blocks) {
#pragma unroll
              for (uint32_t kk = 0; kk < kBlockK / 32; ++kk)
                mma_i8<2>(tmem + b * NT, dw + u * (2 * PairSmem::kHalf >> 4) + kk * 2,
                          dx + u * (2 * PairSmem::kHalf >> 4) + kk * 2, idesc, kb > 0 || u > 0 || kk > 0);
            }
          pair_commit(&sm.empty[s]);
        }
        pair_commit(&sm.acc_full[b]);
      }
      if (any_of(*abort)) break;
    }
  } else {
    // ---- scales and output ----
    const int quarter = warp & 3;
    uint32_t n = 0;
    for (uint64_t tile = first; more; tile += step, more = walk.at(tile, t), ++n) {
      const uint32_t b = n & 1;
      const uint32_t channel = t.channel0 + rank * 128 + quarter * 32 + lane;
      const float sb = P.sb && channel < P.n ? __ldg(P.sb + (uint64_t)t.group * P.n + channel) : 1.0f;
      const uint32_t from = (warp - 2) / 4 * kHalfTokens;
      take_scales(P, t, from, from + kHalfTokens, sm.scales[warp - 2]);
      if (any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort)) {
        *abort = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      put_tile<T>(P, t, tmem + ((uint32_t)(quarter * 32) << 16) + b * NT, channel, sb, from, from + kHalfTokens,
                  sm.scales[warp - 2]);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_remote(remote(sa(&sm.acc_empty[b]), 0));
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cg::this_cluster().sync();
  // A wait gave up in either CTA (its flag is read after both have stopped):
  // what is still in flight ends before shared memory and TMEM are given back.
  const bool stop = *abort || *(volatile int*)cg::this_cluster().map_shared_rank(&sm.abort, rank ^ 1);
  if (stop) {
    if (warp == 0 && elect_one()) {
      atomicOr(P.trap, kDeviceTimeout);
      if (rank == 0)
        for (uint32_t i = it > kPairStages ? it - kPairStages : 0; i < it; ++i)
          mbar_wait(&sm.full[i % kPairStages], (i / kPairStages) & 1, nullptr);
    }
    if (warp == 1 && rank == 0 && elect_one()) {
      pair_commit(&sm.drained);
      mbar_wait(&sm.drained, 0, nullptr);
    }
  }
  __syncwarp();
  cg::this_cluster().sync();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// ---- operands that TMA cannot read ----------------------------------------------------
//
// Bases or strides off 16 bytes: sixteen warps bring a block of k at a time into a
// raw ring with cp.async, as the aligned words of 16 bytes that hold it (nine
// for a row's 128 bytes), and from there shift it into the swizzled layout. A
// row's words are copied and read by the same eight lanes, so a warp waits for
// nobody. Words that do not lie wholly inside the matrix are gathered byte by
// byte. Everything else is as in the kernel of single CTAs.

constexpr int kCopyThreads = 512;  // 4096 x 8192 x 4097: 0.55 ms, with 256 0.71
constexpr int kCopyRows = kCopyThreads / 8;  // at a time
constexpr int kAnyOut = 4;  // warps that write: the copies need the registers

template <int NT, int STAGES>
struct AnySmem {
  static constexpr int kRows = 128 + NT;  // of weights, then of tokens
  static constexpr int kRawRow = 9 * 16;
  uint8_t stage[STAGES][kRows * kBlockK];
  uint8_t raw[STAGES][kRows * kRawRow];
  uint64_t full[STAGES], empty[STAGES];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drained;
  alignas(16) float scales[kAnyOut][kHalfTokens];
  uint32_t tmem_base;
  int abort;
};

struct AnyArgs {
  const int8_t* A;
  const int8_t* B;
  uint64_t lda, ldb, ldg;
  uint64_t a_bytes, b_bytes;  // from the first to the last
  uint32_t k;
};

__device__ __forceinline__ uint4 load16(const uint8_t* p, const uint8_t* lo, const uint8_t* hi) {
  if (p >= lo && p + 16 <= hi) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {};
  for (int i = 0; i < 16; ++i)
    if (p + i >= lo && p + i < hi) w[i / 4] |= (uint32_t)__ldg(p + i) << (8 * (i % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One operand of a tile as a copying thread sees it: 16 bytes of each 128 of
// every kCopyRows-th row, which is a multiple of 16 bytes on whatever the
// stride, so the shift is the same for all of a thread's rows.
struct RowsAt {
  const uint8_t* mine;     // the aligned word of its first row at k = 0
  const uint8_t *lo, *hi;  // the matrix
  uint64_t step;           // kCopyRows rows
  uint32_t rows, k, sh;
  bool low;  // no word of the first block begins before the matrix

  __device__ __forceinline__ void set(const uint8_t* first, uint64_t ld, uint32_t r, uint32_t len, const uint8_t* from,
                                      const uint8_t* to) {
    const uint8_t* p = first + (uint64_t)(threadIdx.x >> 3) * ld + (threadIdx.x & 7) * 16;
    sh = (uint32_t)(uintptr_t)p & 15;
    mine = p - sh;
    lo = from;
    hi = to;
    step = kCopyRows * ld;
    rows = r;
    k = len;
    low = ((uintptr_t)first & 15) == 0 || first - 15 >= from;
  }

  template <int ROWS>
  __device__ __forceinline__ void start(uint8_t* raw, uint32_t k0) const {
    const uint32_t c = threadIdx.x & 7, r0 = threadIdx.x >> 3, at = k0 + c * 16;
    const uint8_t* w = mine + k0;
    uint32_t to = sa(raw + r0 * (9 * 16) + c * 16);
    if (k0 + kBlockK + 16 <= k && (low || k0 > 0)) {
      // every word lies in its row, give or take 15 bytes that the row or the matrix has
#pragma unroll
      for (int i = 0; i < (ROWS + kCopyRows - 1) / kCopyRows; ++i, w += step, to += kCopyRows * 9 * 16)
        if (r0 + i * kCopyRows < rows) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(w) : "memory");
          if (c == 7) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16), "l"(w + 16) : "memory");
        }
    } else {
#pragma unroll 1
      for (int i = 0; i < (ROWS + kCopyRows - 1) / kCopyRows; ++i, w += step, to += kCopyRows * 9 * 16) {
        if (r0 + i * kCopyRows >= rows || at >= k) continue;
        word(to, w);
        // the next lane's word too where that lane has nothing to copy
        if (c == 7 || at + 16 >= k) word(to + 16, w + 16);
      }
    }
  }

  __device__ __forceinline__ void word(uint32_t to, const uint8_t* w) const {
    if (w >= lo && w + 16 <= hi) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(w) : "memory");
    } else {
      const uint4 v = load16(w, lo, hi);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
  }

  template <int ROWS>
  __device__ __forceinline__ void shift(const uint8_t* raw, uint8_t* tile, uint32_t k0) const {
    const uint32_t c = threadIdx.x & 7, r0 = threadIdx.x >> 3, at = k0 + c * 16;
    raw += r0 * (9 * 16) + c * 16;
    tile += r0 * kBlockK + ((c ^ (r0 & 7)) << 4);
    const uint32_t left = k <= at ? 0 : k - at;
#pragma unroll
    for (int i = 0; i < (ROWS + kCopyRows - 1) / kCopyRows; ++i) {
      if (ROWS % kCopyRows && r0 + i * kCopyRows >= ROWS) break;
      const uint4* w = reinterpret_cast<const uint4*>(raw + i * (kCopyRows * 9 * 16));
      uint4 v = straddle(w[0], w[1], sh);
      if (left < 16) {  // zeros behind k
        uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          q[j] = left >= 4 * j + 4 ? q[j] : left <= 4 * j ? 0u : q[j] & ((1u << (8 * (left - 4 * j))) - 1);
        v = make_uint4(q[0], q[1], q[2], q[3]);
      }
      *reinterpret_cast<uint4*>(tile + i * (kCopyRows * kBlockK)) = v;
    }
  }
};

template <typename T, int NT, int STAGES>
__global__ void __launch_bounds__(kCopyThreads + 32 * (1 + kAnyOut), 1)
    mm_i8_any_kernel(const __grid_constant__ AnyArgs Q, const __grid_constant__ TcArgs P) {
  using Smem = AnySmem<NT, STAGES>;
  constexpr uint32_t kCols = 2 * NT;
  constexpr int kOut = kAnyOut, kCopy = kCopyThreads / 32;
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
      mbar_init(&sm.acc_empty[b], kOut);
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
  TileWalk walk{P.offsets, P.groups, P.m, NT, 128, (P.n + 127) / 128, P.trap};
  walk.load();
  Tile t;
  bool more = walk.at(blockIdx.x, t);
  uint32_t it = 0;

  if (warp < kCopy) {
    // ---- copies ----
    const uint8_t *alo = reinterpret_cast<const uint8_t*>(Q.A), *blo = reinterpret_cast<const uint8_t*>(Q.B);
    RowsAt w, x;
    for (uint64_t tile = blockIdx.x; more; tile += gridDim.x, more = walk.at(tile, t)) {
      w.set(blo + t.group * Q.ldg + t.channel0 * Q.ldb, Q.ldb, P.n - t.channel0, Q.k, blo, blo + Q.b_bytes);
      x.set(alo + t.token0 * Q.lda, Q.lda, t.tokens, Q.k, alo, alo + Q.a_bytes);
      auto start = [&](uint32_t kb) {  // one commit group a block, empty past the last
        if (kb < P.k_blocks) {
          uint8_t* raw = sm.raw[kb % STAGES];
          w.start<128>(raw, kb * kBlockK);
          x.start<NT>(raw + 128 * Smem::kRawRow, kb * kBlockK);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll 1
      for (uint32_t kb = 0; kb < STAGES - 1; ++kb) start(kb);
      bool gone = false;
#pragma unroll 1
      for (uint32_t kb = 0; kb < P.k_blocks; ++kb, ++it) {
        start(kb + STAGES - 1);  // its slot was read a turn ago
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        const uint32_t s = it % STAGES;
        gone = !mbar_wait(&sm.empty[s], ((it / STAGES) & 1) ^ 1, abort);
        gone = any_of(gone);  // also: the warp's copies are there for all its lanes
        if (gone) break;
        __syncwarp();
        const uint8_t* raw = sm.raw[kb % STAGES];
        w.shift<128>(raw, sm.stage[s], kb * kBlockK);
        x.shift<NT>(raw + 128 * Smem::kRawRow, sm.stage[s] + 128 * kBlockK, kb * kBlockK);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&sm.full[s]);
        __syncwarp();
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      if (gone) *abort = 1;
      if (any_of(*abort)) break;
    }
  } else if (warp == kCopy) {
    // ---- products ----
    uint32_t n = 0;
    for (uint64_t tile = blockIdx.x; more; tile += gridDim.x, more = walk.at(tile, t), ++n) {
      const uint32_t b = n & 1;
      if (elect_one()) {
        const uint32_t idesc = idesc_i8(128, (int)((t.tokens + 15) / 16 * 16));
        if (!mbar_wait(&sm.acc_empty[b], ((n >> 1) & 1) ^ 1, abort)) *abort = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (uint32_t kb = 0; kb < P.k_blocks && !*abort; ++kb, ++it) {
          const uint32_t s = it % STAGES;
          if (!mbar_wait(&sm.full[s], (it / STAGES) & 1, abort)) {
            *abort = 1;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dw = desc128(sm.stage[s]), dx = desc128(sm.stage[s] + 128 * kBlockK);
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            mma_i8<1>(tmem + b * NT, dw + kk * 2, dx + kk * 2, idesc, kb > 0 || kk > 0);
          mma_commit(&sm.empty[s]);
        }
        mma_commit(&sm.acc_full[b]);
      }
      if (any_of(*abort)) break;
    }
  } else {
    // ---- scales and output ----
    const int quarter = warp & 3, half = (warp - kCopy - 1) / 4;
    constexpr int kShare = NT / (kOut / 4);
    uint32_t n = 0;
    for (uint64_t tile = blockIdx.x; more; tile += gridDim.x, more = walk.at(tile, t), ++n) {
      const uint32_t b = n & 1;
      const uint32_t channel = t.channel0 + quarter * 32 + lane;
      const float sb = P.sb && channel < P.n ? __ldg(P.sb + (uint64_t)t.group * P.n + channel) : 1.0f;
      float* scales = sm.scales[warp - kCopy - 1];
      take_scales(P, t, half * kShare, half * kShare + kShare, scales);
      if (any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort)) {
        *abort = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      put_tile<T>(P, t, tmem + ((uint32_t)(quarter * 32) << 16) + b * NT, channel, sb, half * kShare,
                  half * kShare + kShare, scales);
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

// C where k is 0: zeros times the scales, which may not be finite.
template <typename T>
__global__ void __launch_bounds__(256) mm_i8_empty_kernel(const __grid_constant__ TcArgs P) {
  grid_wait();
  grid_go();
  TileWalk walk{P.offsets, P.groups, P.m, 32, 256, (P.n + 255) / 256, P.trap};
  walk.load();
  Tile t;
  for (uint64_t tile = blockIdx.x; walk.at(tile, t); tile += gridDim.x) {
    const uint32_t j = t.channel0 + threadIdx.x;
    if (j >= P.n) continue;
    const float sb = P.sb ? __ldg(P.sb + (uint64_t)t.group * P.n + j) : 1.0f;
    for (uint32_t i = t.token0; i < t.token0 + t.tokens; ++i)
      static_cast<T*>(P.C)[(uint64_t)i * P.ldc + j] = scaled<T>(0, P.sa ? __ldg(P.sa + i) : 1.0f, sb);
  }
}

// ---- host ----------------------------------------------------------------------------

// rows x k bytes (x matrices) in boxes of 128 bytes x box_rows.
int make_map(CUtensorMap* map, const int8_t* base, uint64_t k, uint64_t rows, uint64_t ld, uint64_t mats, uint64_t ldm,
             int dims, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const uint64_t k16 = (k + 15) & ~15ull;
  // a stride that no access uses (one row, one matrix) may be anything: any valid one stands in
  cuuint64_t dim[3] = {k, rows, mats};
  cuuint64_t stride[2] = {rows > 1 ? ld : k16, mats > 1 ? ldm : (rows > 1 ? ld : k16) * rows};
  cuuint32_t box[3] = {kBlockK, box_rows, 1}, one[3] = {1, 1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, (void*)base, dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return 0;
}

// Whether TMA can read both operands where they lie (k > 0).
bool tma_reads(const MapalI8Site& s, const int8_t* A, const int8_t* B) {
  const uint64_t lim = 1ull << 39;
  const bool a = aligned16(A) && (s.m == 1 || (s.lda % 16 == 0 && s.lda < lim));
  const bool b = aligned16(B) && (s.n == 1 || (s.ldb % 16 == 0 && s.ldb < lim)) &&
                 (s.groups == 1 || (s.ldg % 16 == 0 && s.ldg < lim));
  return a && b && s.n * (s.n == 1 ? s.k : s.ldb) < lim;
}

// A way to cut the product: channels and tokens of a tile, parts of k; pairs
// of CTAs have 256 channels.
struct Cut {
  uint32_t channels, tokens, split;
};

// Tiles of a cut: at most one part-filled token tile for each group with rows
// (the offsets are on the device).
uint64_t tiles_of(const MapalI8Site& s, bool grouped, const Cut& c) {
  const uint64_t with_rows = s.groups < s.m ? s.groups : s.m;
  const uint64_t token_tiles = grouped ? s.m / c.tokens + with_rows : (s.m + c.tokens - 1) / c.tokens;
  return token_tiles * ((s.n + c.channels - 1) / c.channels);
}

// Cycles of a cut, from what bounds its tiles: the MMA (N/2 cycles for 128
// channels and 32 bytes of k, 32 + N/4 at least), and the loads, at up to 64 bytes a
// cycle for an SM and 6200 for all. Tiles run in waves, each with a start and
// an end that nothing overlaps when it is the only one. It ranks cuts; as a time
// it is short where pairs have one wave, whose output of 256 x 256 nothing hides
// (at 1.9 GHz against measured, n 8192, k 4096: 256 tokens 9.4 and 17.1 us, 512
// 12.2 and 17.7, 1024 27.9 and 28.7, 2048 56 and 50). 64 of 148 SMs work on 256.
double cycles_of(const MapalI8Site& s, bool grouped, const Cut& c, int sms) {
  const bool pair = c.channels == 256;
  const double tiles = (double)tiles_of(s, grouped, c) * c.split, at_once = pair ? sms / 2 : sms;
  const double active = tiles < at_once ? tiles : at_once, ctas = pair ? 2 * active : active;
  const double k_blocks = (double)((s.k + kBlockK - 1) / kBlockK) / c.split;
  const double rate = 6200.0 / ctas < 64.0 ? 6200.0 / ctas : 64.0;
  const double load = (pair ? 256 : c.channels + c.tokens) * (double)kBlockK / rate;
  const double tokens = s.m < c.tokens ? (double)((s.m + 15) / 16 * 16) : c.tokens;
  const double mma = 4 * (tokens / 4 + 32 > tokens / 2 ? tokens / 4 + 32 : tokens / 2);
  const double waves = (double)(uint64_t)((tiles + at_once - 1) / at_once);
  return waves * (k_blocks * (load > mma ? load : mma) + 1500) + (c.split > 1 ? 5500 : 0);
}

// B as [group][eight channels][block of k][8][128 bytes], in boxes of
// channels/8 x blocks.
int make_folded_map(CUtensorMap* map, const MapalI8Site& s, const int8_t* B, uint32_t channels, uint32_t blocks) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dim[5] = {(cuuint64_t)kBlockK, 8, s.k / kBlockK, s.n / 8, s.groups};
  cuuint64_t stride[4] = {s.ldb, (cuuint64_t)kBlockK, 8 * s.ldb, s.groups > 1 ? s.ldg : s.n * s.ldb};
  cuuint32_t box[5] = {(cuuint32_t)kBlockK, 8, blocks, channels / 8, 1}, one[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, (void*)B, dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return 0;
}

int launch_maps(const MapalI8Site& s, const int8_t* A, const int8_t* B, uint32_t channels, uint32_t tokens,
                uint32_t folded, CUtensorMap* mw, CUtensorMap* mx) {
  if (folded)
    MAPAL_TRY(make_folded_map(mw, s, B, channels, folded));
  else
    MAPAL_TRY(make_map(mw, B, s.k, s.n, s.ldb, s.groups, s.ldg, 3, channels));
  return make_map(mx, A, s.k, s.m, s.lda, 1, 0, 2, tokens);
}

template <typename T, int NT, int CH, int KB, int STAGES>
int launch_tc(const DeviceSlot& D, const MapalI8Site& s, const int8_t* A, const int8_t* B, TcArgs P, uint64_t tiles) {
  using Smem = TcSmem<NT, CH, KB, STAGES>;
  CUtensorMap mw, mx;
  P.folded = s.k % kBlockK == 0 && s.n % 8 == 0 && s.ldb < (1ull << 36);
  MAPAL_TRY(launch_maps(s, A, B, CH, NT, P.folded ? KB : 0, &mw, &mx));
  constexpr size_t most = sizeof(Smem) + 1024 + (NT <= 64 ? NT * CH * 4 : 0);
  static_assert(most <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  auto kernel = mm_i8_tc_kernel<T, NT, CH, KB, STAGES>;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, most, "matmul_i8 shared memory"));
  const uint64_t cap = P.split > 1 ? tiles : (uint64_t)D.prof.sm_count;
  return launch_rows(kernel, (unsigned)((tiles < cap ? tiles : cap) * P.split), 64 + 32 * out_warps(NT),
                     sizeof(Smem) + 1024 + (P.split > 1 ? NT * CH * 4 : 0), D.stream, P.split, mw, mx, P);
}

template <typename T>
int launch_pair(const DeviceSlot& D, const MapalI8Site& s, const int8_t* A, const int8_t* B, const TcArgs& P,
                uint64_t tiles) {
  CUtensorMap mw, mx;
  MAPAL_TRY(launch_maps(s, A, B, 128, 128, 0, &mw, &mx));
  constexpr size_t smem = sizeof(PairSmem) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  MAPAL_TRY(ensure_smem_attr(done, (const void*)mm_i8_pair_kernel<T>, D.device, smem, "matmul_i8 shared memory"));
  const uint64_t cap = D.prof.sm_count / 2;
  return launch_rows(mm_i8_pair_kernel<T>, (unsigned)((tiles < cap ? tiles : cap) * 2), 64 + 32 * out_warps(256), smem,
                     D.stream, 1, mw, mx, P);
}

template <typename T, int NT, int STAGES>
int launch_any(const DeviceSlot& D, const MapalI8Site& s, const int8_t* A, const int8_t* B, const TcArgs& P,
               uint64_t tiles) {
  constexpr size_t smem = sizeof(AnySmem<NT, STAGES>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  auto kernel = mm_i8_any_kernel<T, NT, STAGES>;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, smem, "matmul_i8 shared memory"));
  const uint64_t one = (s.n - 1) * s.ldb + s.k;
  const AnyArgs q{A, B, s.lda, s.ldb, s.ldg, (s.m - 1) * s.lda + s.k, (s.groups - 1) * s.ldg + one, (uint32_t)s.k};
  const uint64_t cap = D.prof.sm_count;
  return launch_rows(kernel, (unsigned)(tiles < cap ? tiles : cap), kCopyThreads + 32 * (1 + kAnyOut), smem, D.stream, 1, q,
                     P);
}

template <typename T>
int run(const DeviceSlot& D, const MapalI8Site& s, const int8_t* A, const float* sa, const int8_t* B, const float* sb,
           const int32_t* offsets, void* C) {
  TcArgs P{};
  P.offsets = offsets;
  P.sa = sa;
  P.sb = sb;
  P.C = C;
  P.trap = D.trap;
  P.ldc = s.ldc;
  P.m = (uint32_t)s.m;
  P.n = (uint32_t)s.n;
  P.groups = s.groups;
  P.k_blocks = (uint32_t)((s.k + kBlockK - 1) / kBlockK);

  if (s.k == 0) {
    const uint64_t tiles = tiles_of(s, offsets, {256, 32, 1}), cap = 8ull * D.prof.sm_count;
    return launch_rows(mm_i8_empty_kernel<T>, (unsigned)(tiles < cap ? tiles : cap), 256, 0, D.stream, 1, P);
  }
  if (!tma_reads(s, A, B)) {
    // the rows that an SM brings for a block of k, over its waves of tiles (81 x
    // 2299 x 1073: 19.7 us with 18 tiles of 128 tokens, 14.1 with 54 of 32, both
    // with 256 copying threads)
    const uint64_t few = tiles_of(s, offsets, {128, 32, 1}), wide = tiles_of(s, offsets, {128, 128, 1});
    const uint64_t sms = D.prof.sm_count;
    if ((few + sms - 1) / sms * (128 + 32) <= (wide + sms - 1) / sms * (128 + 128)) return launch_any<T, 32, 5>(D, s, A, B, P, few);
    return launch_any<T, 128, 3>(D, s, A, B, P, wide);
  }
  static constexpr Cut kCuts[] = {{256, 256, 1}, {128, 128, 1}, {64, 128, 1}, {128, 64, 1}, {64, 64, 1},
                                  {128, 32, 1},  {64, 32, 1},   {128, 16, 1}, {64, 16, 1},  {32, 16, 1}};
  Cut best{};
  double least = 0;
  for (Cut c : kCuts)
    for (c.split = 1; c.split <= 8; c.split *= 2) {
      if (c.split > 1 && (c.tokens > 64 || c.split * 4 > P.k_blocks ||
                          tiles_of(s, offsets, c) * c.split > (uint64_t)D.prof.sm_count))
        break;
      const double cy = cycles_of(s, offsets, c, D.prof.sm_count);
      if (best.channels == 0 || cy < least) {
        best = c;
        least = cy;
      }
    }
  P.split = best.split;
  const uint64_t tiles = tiles_of(s, offsets, best);
  switch (best.channels * 1000 + best.tokens) {
    case 256256: return launch_pair<T>(D, s, A, B, P, tiles);
    case 128128: return launch_tc<T, 128, 128, 2, 3>(D, s, A, B, P, tiles);
    case 64128: return launch_tc<T, 128, 64, 2, 4>(D, s, A, B, P, tiles);
    case 128064: return launch_tc<T, 64, 128, 2, 3>(D, s, A, B, P, tiles);
    case 64064: return launch_tc<T, 64, 64, 2, 6>(D, s, A, B, P, tiles);
    case 128032: return launch_tc<T, 32, 128, 2, 5>(D, s, A, B, P, tiles);
    case 64032: return launch_tc<T, 32, 64, 4, 4>(D, s, A, B, P, tiles);
    case 128016: return launch_tc<T, 16, 128, 2, 5>(D, s, A, B, P, tiles);
    case 64016: return launch_tc<T, 16, 64, 4, 4>(D, s, A, B, P, tiles);
    default: return launch_tc<T, 16, 32, 4, 7>(D, s, A, B, P, tiles);
  }
}

int check_site(const MapalI8Site* s) {
  if (!s) return set_error(MAPAL_ERR_INVALID, "site is null");
  const int es = dtype_bytes(s->dtype);
  if (es < 2) return set_error(MAPAL_ERR_INVALID, "C is f32, f16 or bf16");
  if (s->groups == 0 || s->groups > 65535) return set_error(MAPAL_ERR_INVALID, "1 to 65535 groups");
  if (s->k >= 131072) return set_error(MAPAL_ERR_UNSUPPORTED, "k of 131072 or more: a sum could leave 32 bits");
  // a tile's last row or channel is counted in 32 bits
  if (s->m > 0x7fffff00ull || s->n > 0x7fffff00ull) return set_error(MAPAL_ERR_UNSUPPORTED, "m or n over 2^31 - 256");
  if (!rows_ok(s->m, s->k, s->lda, 1) || !rows_ok(s->n, s->k, s->ldb, 1) || !rows_ok(s->m, s->n, s->ldc, es))
    return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
  const uint64_t one = s->n ? (s->n - 1) * s->ldb + s->k : 0;
  if (s->groups > 1 && !rows_ok(s->groups, one, s->ldg, 1))
    return set_error(MAPAL_ERR_INVALID, "the stride between groups is shorter than a matrix, or too long");
  return 0;
}

}  // namespace

extern "C" int mapal_gpu_matmul_i8(MapalGpuCtx* ctx, const MapalI8Site* site, const int8_t* A, const float* scale_a,
                                   const int8_t* B, const float* scale_b, const int32_t* offsets, void* C) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site));
    const MapalI8Site& s = *site;
    if (!offsets && s.groups != 1) return set_error(MAPAL_ERR_INVALID, "several groups need offsets");
    if (s.m == 0 || s.n == 0) return 0;
    if (!C || (s.k && (!A || !B))) return set_error(MAPAL_ERR_INVALID, "null A, B or C");
    const int es = dtype_bytes(s.dtype);
    if (((uintptr_t)C & (es - 1)) || ((uintptr_t)scale_a & 3) || ((uintptr_t)scale_b & 3) || ((uintptr_t)offsets & 3))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    auto go = [&](auto t) {
      using T = decltype(t);
      return run<T>(D, s, A, scale_a, B, scale_b, offsets, C);
    };
    MAPAL_TRY(s.dtype == MAPAL_DTYPE_F32   ? go(float{})
              : s.dtype == MAPAL_DTYPE_F16 ? go(__half{})
                                           : go(__nv_bfloat16{}));
    return finish(ctx, 0, true);
  });
}

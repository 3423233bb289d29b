// product.cuh — products in 16-bit floats on the tensor cores: what the products
// by expert (product.cu) and the loss (linear_loss.cu) share. Not part of the ABI.
//
// Three products of the same arrays X (m x k), W (groups of n x k) and Y or dY
// (m x n), with rows of X and Y sorted by group:
//   forward   Y[i] = W[g] X[i]          sums over k
//   grad x    dX[i] = W[g]^T dY[i]      sums over n
//   grad w    dW[g] = sum_i dY[i]^T X[i]  sums over the rows of g
// Each is D[lane][col] = sum_t A[lane][t]*B[col][t] in a tile of tensor memory,
// with the dimension along which the output is contiguous on the lanes (n, k, k),
// so that neighbouring lanes hold neighbouring elements, and the output's rows on
// the columns (rows, rows, n). An operand whose memory runs along t is K-major, one
// whose memory runs along its lanes or columns MN-major; the tensor cores take both
// at the same rate, so no operand is ever transposed in memory:
//               A            B
//   forward   W K-major    X  K-major
//   grad x    W MN-major   dY K-major
//   grad w    X MN-major   dY MN-major
// Products of 16-bit values are exact in f32, sums are f32 in tensor memory,
// rounded once on writing.
#pragma once

#include <cooperative_groups.h>

#include "tiles.cuh"

enum ProductMode { kForward = 0, kGradX = 1, kGradW = 2 };

constexpr int kStepK = 64;  // elements of t in a block: 128 bytes, the swizzle's width

struct ProductArgs {
  const int32_t* offsets;  // null: one group of all rows
  unsigned* trap;
  uint32_t groups, m;
  uint32_t lanes;  // extent of the lanes' dimension
  const int32_t* lane_count;  // where not null: how many of them count, on the device
  uint32_t cols;   // grad w: extent of the columns' dimension (n)
  uint32_t depth;  // forward, grad x: extent of t
  uint32_t parts;  // forward, grad x: t cut into so many parts, each with its own output
  uint32_t bf16;
  uint32_t box;  // pairs, forward: lanes that a CTA loads, see launch_product_pair
};

struct Job {
  uint32_t group, col0, cols, lane0;
  uint32_t t0, depth;  // the range of t
  uint32_t part;
};

// A warp's walk over every step-th job of tiles of NT columns and CH lanes; every
// lane gets the answers. Lanes run fastest, so that the tiles in flight share their
// columns' operand. Divisions are made once: one by one, the 64-bit ones of a tile's
// number took a lone warp 1200 cycles a tile, as long as four blocks' products.
template <int MODE, int NT, int CH>
struct JobWalk {
  const ProductArgs& P;
  TileWalk tiles;
  uint32_t lane_tiles, per_part;
  uint64_t outer;               // column tiles (forward, grad x: of all parts) before this one
  uint32_t inner;               // its lane tile
  uint64_t d_outer;             // of a step
  uint32_t d_inner;
  uint32_t col_tiles, col, group, d_col, d_group;  // grad w: outer, divided by the column tiles of a matrix
  uint32_t lo, hi;

  __device__ JobWalk(const ProductArgs& p, uint64_t first, uint64_t step) : P(p) {
    uint32_t lanes = p.lanes;
    if (p.lane_count) lanes = min(lanes, (uint32_t)max(__ldg(p.lane_count), 0));
    lane_tiles = (lanes + CH - 1) / CH;
    const uint32_t by = max(lane_tiles, 1u);
    if (((first | step) >> 32) == 0) {
      outer = (uint32_t)first / by;
      d_outer = (uint32_t)step / by;
    } else {
      outer = first / by;
      d_outer = step / by;
    }
    inner = (uint32_t)(first - outer * by);
    d_inner = (uint32_t)(step - d_outer * by);
    if constexpr (MODE == kGradW) {
      // at most 2^32 column tiles of all matrices: 65535 of 2^23
      col_tiles = (p.cols + NT - 1) / NT;
      group = (uint32_t)(outer / col_tiles);
      col = (uint32_t)(outer - (uint64_t)group * col_tiles);
      d_group = (uint32_t)(d_outer / col_tiles);
      d_col = (uint32_t)(d_outer - (uint64_t)d_group * col_tiles);
      range();
    } else {
      tiles = TileWalk{p.offsets, p.groups, p.m, NT, CH, lane_tiles, p.trap};
      tiles.load();
      const uint32_t blocks = (p.depth + kStepK - 1) / kStepK;
      per_part = p.parts > 1 ? (blocks + p.parts - 1) / p.parts * kStepK : p.depth;
    }
  }

  // grad w: the group's rows.
  __device__ __forceinline__ void range() {
    lo = 0, hi = P.m;
    if (P.offsets && group < P.groups) {
      const int32_t a = __ldg(P.offsets + group), b = __ldg(P.offsets + group + 1);
      const bool bad = a < 0 || b < a || (uint32_t)b > P.m;
      if (bad && (threadIdx.x & 31) == 0) atomicMax(P.trap, kTrapOob);
      lo = min((uint32_t)max(a, 0), P.m);
      hi = max(lo, min((uint32_t)max(b, 0), P.m));
    }
  }

  __device__ __forceinline__ bool now(Job& j) {
    if (lane_tiles == 0) return false;
    j.lane0 = inner * CH;
    j.part = 0;
    if constexpr (MODE == kGradW) {
      if (group >= P.groups) return false;
      j.group = group;
      j.col0 = col * NT;
      j.cols = min((uint32_t)NT, P.cols - j.col0);
      j.t0 = lo;
      j.depth = hi - lo;
    } else {
      // parts (of one group of all rows) run slowest: the tiles of one share the operands' blocks
      uint64_t at = outer;
      if (P.parts > 1) {
        if (at >= (uint64_t)tiles.chunk * P.parts) return false;
        j.part = (uint32_t)(at / tiles.chunk);
        at -= (uint64_t)j.part * tiles.chunk;
      }
      Tile t;
      if (!tiles.find(at, t)) return false;
      j.group = t.group;
      j.col0 = t.token0;
      j.cols = t.tokens;
      j.t0 = min(j.part * per_part, P.depth);
      j.depth = min(per_part, P.depth - j.t0);
    }
    return true;
  }

  __device__ __forceinline__ bool next(Job& j) {
    inner += d_inner;
    const uint32_t carry = inner >= lane_tiles;
    inner -= carry ? lane_tiles : 0;
    if constexpr (MODE == kGradW) {
      col += d_col + carry;
      uint32_t g = group + d_group;
      if (col >= col_tiles) {
        col -= col_tiles;
        ++g;
      }
      if (g != group) {
        group = g;
        range();
      }
    } else {
      outer += d_outer + carry;
    }
    return now(j);
  }
};

// ---- tensor core pieces --------------------------------------------------------------

// MN-major, 128-byte swizzle: 64 elements along the lanes or columns by 8 steps of t
// in 1024 bytes; the next 8 steps follow, the next 64 elements lie `chunk` bytes on.
__device__ __forceinline__ uint64_t desc_mn(const void* p, uint32_t chunk) {
  return (uint64_t)((sa(p) & 0x3FFFFu) >> 4) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(const void* p) {
  return MN ? desc_mn(p, kStepK * 128) : desc128(p);
}
// 16 steps of t on, in units of 16 bytes: 32 bytes of a K-major row, 16 rows of an MN-major one.
template <bool MN>
__device__ __forceinline__ constexpr uint32_t operand_step() {
  return MN ? 16 * 128 / 16 : 2;
}

// D f32, A and B both f16 or both bf16.
template <int MODE>
__device__ __forceinline__ uint32_t idesc_f16(uint32_t bf16, int m, int n) {
  return (1u << 4) | (bf16 << 7) | (bf16 << 10) | ((MODE != kForward ? 1u : 0u) << 15) |
         ((MODE == kGradW ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&f)[16]) {
  int r[16];
  tmem_ld16(taddr, r);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __int_as_float(r[i]);
}

// ---- writing a tile --------------------------------------------------------------------

// Sixteen columns of 32 lanes, one a lane, to 16 rows of memory: one conversion for two.
template <typename T>
__device__ __forceinline__ void put16(T* c, uint64_t ld, const float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float v[4] = {f[i], f[i + 1], f[i + 2], f[i + 3]};
    Pack<T, 4> o;
    o.set(v);
    T w[4];
    memcpy(w, o.w, sizeof(w));
    c[0] = w[0];
    c[ld] = w[1];
    c[2 * ld] = w[2];
    c[3 * ld] = w[3];
    c += 4 * ld;
  }
}

// 16 lanes by 32 columns of tensor memory as fragments: of every 8 columns a thread
// gets two neighbours of lane t/4 and the same of lane t/4 + 8.
__device__ __forceinline__ void tmem_ld16x32(uint32_t taddr, float (&f)[16]) {
  int r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __int_as_float(r[i]);
}

constexpr int kOutScratch = 32 * 64;  // bytes of shared memory that a writing warp needs
constexpr int kTurnCols = 32;  // columns of tensor memory that it reads at a time, whatever is left of the tile

// Columns [from, to) of a warp's 32 lanes, of which `left` exist, as 16-bit values: 32
// columns at a time are turned in shared memory (stmatrix, transposed) so that a
// thread writes 8 lanes of a column at once, row(j) + 8*its part; every row is
// 16-byte aligned. Elements written one by one keep a warp 32 stores for what
// takes 4 here (the weights' gradient of 256 rows over 64 matrices of 1024 x 2048,
// which is writing: 76 us with them, 69 with these).
template <typename T, bool SCALE, typename Row>
__device__ __forceinline__ void put_turned(uint32_t taddr, uint32_t from, uint32_t to, int left, bool zero, float factor,
                                           uint8_t* scratch, Row&& row) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t put = sa(scratch) + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
  const uint32_t get = (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
  const int have = left - (int)(lane & 3) * 8;  // of this thread's 8 lanes
  float f[2][16];
  auto load = [&](uint32_t j0) {
    tmem_ld16x32(taddr + j0, f[0]);
    tmem_ld16x32(taddr + (16u << 16) + j0, f[1]);
  };
  if (zero) {  // sums over nothing
    for (uint32_t j0 = from; j0 < to; j0 += 8) {
      const uint32_t col = j0 + (lane >> 2);
      if (col < to)
        for (int e = 0; e < min(8, have); ++e) row(col)[(lane & 3) * 8 + e] = from_f32<T>(0.0f);
    }
    return;
  }
  if (from < to) load(from);
  for (uint32_t j0 = from; j0 < to; j0 += kTurnCols) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(f[0][i]), "+f"(f[1][i]));
    uint32_t w[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // lanes t/4 and t/4 + 8 of both halves
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = SCALE ? f[h][4 * q + e] * factor : f[h][4 * q + e];
        Pack<T, 4> o;
        o.set(v);
        w[q][2 * h] = o.w[0], w[q][2 * h + 1] = o.w[1];
      }
    if (j0 + kTurnCols < to) load(j0 + kTurnCols);  // beside the stores
#pragma unroll
    for (int q = 0; q < 4; ++q)
      asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(put + q * 512),
                   "r"(w[q][0]), "r"(w[q][1]), "r"(w[q][2]), "r"(w[q][3])
                   : "memory");
    __syncwarp();
    Pack<T, 8> o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(scratch + i * 512 + get);
      o[i].w[0] = v.x, o[i].w[1] = v.y, o[i].w[2] = v.z, o[i].w[3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t col = j0 + i * 8 + (lane >> 2);
      if (col < to && have > 0) {
        T* c = row(col) + (lane & 3) * 8;
        if (have >= 8)
          *reinterpret_cast<Pack<T, 8>*>(c) = o[i];
        else
          st_part(c, o[i], (1u << have) - 1);
      }
    }
    __syncwarp();
  }
}

// The output as it lies in memory: column j of a job at row (grad w: row of the
// group's matrix), lanes along the row. wide: 16-bit rows on 16-byte boundaries.
template <int MODE, typename T>
struct StoreTile {
  static constexpr int kRun = 0;  // see the pair of CTAs
  T* out;
  uint64_t ld, ldg;  // rows, groups' matrices
  bool wide;

  __device__ __forceinline__ T* at(const Job& j, uint32_t lane0) const {
    return out + (MODE == kGradW ? (uint64_t)j.group * ldg : 0) + (uint64_t)j.col0 * ld + lane0;
  }

  // Columns [from, to) of the 32 lanes of a warp from lane0 on.
  __device__ __forceinline__ void put(const ProductArgs& P, const Job& j, uint32_t taddr, uint32_t lane0, uint32_t from,
                                      uint32_t to, uint8_t* scratch) const {
    if constexpr (sizeof(T) == 2) {
      if (wide) {
        T* c = at(j, lane0);
        put_turned<T, false>(taddr, from, min(to, j.cols), (int)(P.lanes - lane0), j.depth == 0, 1.0f, scratch,
                             [&](uint32_t col) { return c + col * ld; });
        return;
      }
    }
    put_plain(P, j, taddr, lane0, from, to);
  }

  // The same, element by element.
  __device__ __forceinline__ void put_plain(const ProductArgs& P, const Job& j, uint32_t taddr, uint32_t lane0,
                                            uint32_t from, uint32_t to) const {
    const bool zero = j.depth == 0;
    to = min(to, j.cols);
    T* c = at(j, lane0);
    const uint32_t lane = threadIdx.x & 31;
    const bool in = lane0 + lane < P.lanes;
    c += from * ld + (in ? lane : 0);
    for (uint32_t j0 = from; j0 < to; j0 += 16, c += 16 * ld) {
      float f[16];
      tmem_ld16f(taddr + j0, f);
      if (zero) {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = 0.0f;
      }
      if (j0 + 16 <= to) {
        if (in) put16(c, ld, f);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (in && j0 + i < to) c[i * ld] = from_f32<T>(f[i]);
      }
    }
  }
};

// ---- a pair of CTAs a tile ---------------------------------------------------------------
//
// 256 lanes by up to 256 columns: each CTA of the pair loads its 128 lanes of A and
// half of B's columns, and the pair's MMA (cta_group::2, issued by the first CTA)
// reads both halves from both, so a CTA moves 32 KB a block of t where a 128 x 256
// tile of its own moves 48. Persistent; two accumulators in tensor memory, so that
// a tile's output runs beside the next one's products.
//
// grad w: the last block of a group's rows may hold rows of the next group. Such a
// block is counted by a barrier of its own (landed); a warp clears the rows behind
// the group's last up to the next 16 (the MMA's step) in both operands, since zero
// times NaN is not zero, and lets the products go on (fixed).
//
// Where the sum's own error counts (Out::kRun, blocks), t is taken in runs: each run's
// sums start from zero in tensor memory, where every step cuts what it adds up, and
// the output warps add the runs up in registers, rounded.
//
// Bound by the tensor cores: 4096^3 bf16 in 95 us (1.45 PFLOP/s, cuBLAS 93), 16384 rows
// of 16 matrices of 4096 x 4096 in 411, 475 and 415 us (1.16 to 1.34 PFLOP/s, at the
// power limit). A tile of 16 blocks has 5 us of start and end around 4 of products.
//
// An operand off 16 bytes (CA, CB) comes by TMA all the same, raw: every eighth of its
// rows lies 16-byte aligned from the one before, so eight maps, one for each row
// number's remainder, each with its base rounded down, bring lines with up to 14
// foreign bytes before them. Copying warps shift them into the swizzled layout:
// a line's remainder, and so its shift, is the same for all of a thread's lines.
// Everything else is as with operands in place. A copy loop through registers
// instead (two aligned words a thread, a block ahead) took 3300 ns a block of
// both operands, waiting for L1's few lines; this takes 770, and 550 where one
// is copied (4096 x 4096 x 4097: 204 us forward, 137 and 152 for the gradients; the
// products alone take 270 a block; with two groups of warps 212 us). Shared memory bounds it: two reads and a write of every
// 16 bytes, 384 cycles an operand's block.

constexpr int kPairTokens = 256, kPairOut = 8;
constexpr int kCopyGroups = 3, kCopyWarps = 4;  // groups of so many warps take turns at the blocks
constexpr uint32_t kToldBytes = 16;
constexpr uint64_t kRawLandNs = 1000000;  // after a wait gave up: for copies in flight that nothing waits for
constexpr int kLineK = 144, kLineMN = 272;  // raw bytes of a line: 64 steps, or 128 lanes or columns, and 16 more
constexpr int kRawOperand = 128 * kLineK;
static_assert(64 * kLineMN <= kRawOperand, "raw lines");

// STAGES of KB blocks; RAW: raw operands side by side in flight.
template <int STAGES, int KB, int RAW>
struct PairSmem {
  static constexpr int kHalf = 128 * 128;  // bytes of a block of lanes, and of columns
  uint8_t stage[STAGES][KB * 2 * kHalf];
  alignas(128) uint8_t raw[RAW == 0 ? 1 : RAW][RAW == 0 ? 16 : kRawOperand];
  uint64_t full[STAGES];    // the first CTA's: both CTAs' loads have landed, their copies are written
  uint64_t empty[STAGES];   // each CTA's own
  uint64_t landed[STAGES];  // each CTA's own: a last block to clear
  uint64_t fixed[STAGES];   // the first CTA's: cleared in both
  uint64_t raw_full[RAW == 0 ? 1 : RAW], raw_empty[RAW == 0 ? 1 : RAW];  // each CTA's own
  uint64_t acc_full[2];     // each CTA's own
  uint64_t acc_empty[2];    // the first CTA's: both CTAs have read the accumulator
  uint64_t drained;
  alignas(16) uint8_t scratch[kPairOut][kOutScratch];
  alignas(16) uint8_t told[kCopyGroups * kCopyWarps + 1][kToldBytes];  // where tell_written's copies go, a warp's each
  uint32_t tmem_base;
  int abort;
};
template <bool CA, bool CB>
struct PairCut {
  static constexpr bool kCopy = CA || CB;
  static constexpr int kStages = kCopy && !(CA && CB) ? 4 : 3, kKB = kCopy ? 1 : 2;
  static constexpr int kRaw = CA && CB ? 3 : kCopy ? 4 : 0;  // raw blocks
  using Smem = PairSmem<kStages, kKB, kRaw * (CA + CB)>;
  static constexpr size_t kSmem = sizeof(Smem) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
};
// loads, products, output, grad w: clearing, and copies
__host__ __device__ constexpr int pair_fixers(int mode, bool ca, bool cb) { return mode == kGradW && !(ca && cb) ? 1 : 0; }
__host__ __device__ constexpr int pair_threads(int mode, bool ca, bool cb) {
  return 64 + 32 * kPairOut + 32 * pair_fixers(mode, ca, cb) + (ca || cb ? 32 * kCopyGroups * kCopyWarps : 0);
}

struct RawMaps {
  CUtensorMap m[8];
};
// A copied operand beside its maps: where row 0 begins in an aligned word and what a row adds.
struct RawPlace {
  uint32_t base, ld;  // bytes, modulo 16
  uint32_t rows;      // from one matrix to the next
};

// Raw lines of the 128 (K-major: rows from row0 on, steps from x on) or 64 (MN-major:
// steps from row0 on, 128 lanes or columns from x on) rows of a block.
template <bool MN>
__device__ __forceinline__ void raw_load(uint8_t* raw, const RawMaps& maps, uint32_t row0, int x, uint64_t* bar) {
  constexpr int kRows = MN ? 8 : 16, kLine = MN ? kLineMN : kLineK;
  mbar_expect_tx(bar, 8 * kRows * kLine);
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i)  // the first rows of each remainder: row0 + i
    tma_load_2d(raw + ((row0 + i) & 7) * (kRows * kLine), &maps.m[(row0 + i) & 7], x, (int)((row0 + i) >> 3), bar);
}

// A thread's share of shifting a raw block into the swizzled layout: 16 bytes of every
// 16th line. left: rows of the block that exist (MN-major; the others become zeros).
template <bool MN>
__device__ __forceinline__ void raw_shift(uint32_t thread, const uint8_t* raw, const RawPlace& o, uint32_t row0, uint32_t lines,
                                          uint32_t left, uint8_t* tile) {
  constexpr int kRows = MN ? 8 : 16, kLine = MN ? kLineMN : kLineK;
  constexpr int kApart = kCopyWarps * 4;  // lines from one turn to the next
  static_assert(kApart == 16, "whole eights of lines, four turns a chunk of 64");
  const uint32_t c = thread & 7, line = thread >> 3;
  const uint32_t sh = (o.base + (row0 + line) * o.ld) & 15;
  const uint32_t s = (row0 + line) & 7, q = (line - ((s - row0) & 7)) >> 3;
  const uint8_t* from = raw + (s * kRows + q) * kLine + c * 16;
  uint8_t* to = tile + line * 128 + ((c ^ (line & 7)) << 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t at = MN ? (i & 3) * 2 * kLine + (i >> 2) * 128 : i * 2 * kLine;
    if (!MN && line + i * kApart >= lines) break;
    uint4 v = straddle(*reinterpret_cast<const uint4*>(from + at), *reinterpret_cast<const uint4*>(from + at + 16), sh);
    if (MN && line + (i & 3) * kApart >= left) v = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(to + i * (kApart * 128)) = v;
  }
}

// An arrival at another CTA's barrier that orders nothing but the tensor memory read
// before it (tcgen05.fence): a release would first wait for the tile's stores.
__device__ __forceinline__ void arrive_remote_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Tells the first CTA's barrier that this warp has written to its own CTA's shared memory,
// `written` among it, which the pair's MMA reads from both CTAs; every writing lane has made
// its part visible to the asynchronous proxy before. The second CTA tells it by a copy of
// 16 bytes between the CTAs: the copy follows what was written, and its completion is a
// release among the CTAs, which a thread's own arrival can be too, but for 500 to 1800
// cycles in which the thread waits for its SM's stores (4096 x 4096 x 4097: 275 us). The
// first CTA's arrival expects the bytes.
__device__ __forceinline__ void tell_written(uint64_t* bar, const void* written, const void* to, uint32_t rank) {
  if (rank == 0)
    mbar_expect_tx(bar, kToldBytes);
  else
    asm volatile(
        "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(remote(sa(to), 0)),
        "r"(sa(written)), "r"(kToldBytes), "r"(remote(sa(bar), 0))
        : "memory");
}

__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(sa(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pair_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(sa(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// A CTA's 128 lanes and its half of the columns of one block of t, of the operands
// that TMA reads. W's map has the groups as its third dimension.
template <int MODE, bool TA, bool TB>
__device__ __forceinline__ void pair_load_block(uint8_t* a, uint8_t* b, const CUtensorMap* map_a, const CUtensorMap* map_b, const Job& j,
                                                int t, int lane0, int col0, bool any_a, uint32_t bar) {
  constexpr int kChunk = kStepK * 128;  // 64 lanes or columns of an MN-major block
  if constexpr (TA) {
    if constexpr (MODE == kForward) {
      if (any_a) pair_load_3d(a, map_a, t, lane0, (int)j.group, bar);
    } else if constexpr (MODE == kGradX) {
      pair_load_3d(a, map_a, lane0, t, (int)j.group, bar);
      pair_load_3d(a + kChunk, map_a, lane0 + 64, t, (int)j.group, bar);
    } else {
      pair_load_2d(a, map_a, lane0, t, bar);
      pair_load_2d(a + kChunk, map_a, lane0 + 64, t, bar);
    }
  }
  if constexpr (TB) {
    if constexpr (MODE == kGradW) {
      pair_load_2d(b, map_b, col0, t, bar);
      pair_load_2d(b + kChunk, map_b, col0 + 64, t, bar);
    } else {
      pair_load_2d(b, map_b, t, col0, bar);
    }
  }
}

// CA, CB: the operand is copied.
template <int MODE, bool CA, bool CB, typename Out>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair_threads(MODE, CA, CB), 1)
    product_pair_kernel(const __grid_constant__ std::conditional_t<CA, RawMaps, CUtensorMap> maps_a,
                        const __grid_constant__ std::conditional_t<CB, RawMaps, CUtensorMap> maps_b, const RawPlace place_a,
                        const RawPlace place_b, const __grid_constant__ ProductArgs P, const __grid_constant__ Out out) {
  namespace cg = cooperative_groups;
  using Cut = PairCut<CA, CB>;
  using Smem = typename Cut::Smem;
  constexpr int NT = kPairTokens, kStages = Cut::kStages, kKB = Cut::kKB, kRaw = Cut::kRaw;
  constexpr bool TA = !CA, TB = !CB;
  constexpr int kFixer = 2 + kPairOut, kCopier = kFixer + pair_fixers(MODE, CA, CB);  // warps
  constexpr bool MA = MODE != kForward, MB = MODE == kGradW;  // MN-major
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t rank = blockIdx.x & 1;
  const uint64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
  volatile int* abort = &sm.abort;
  auto give_up = [&]() {  // both CTAs stop
    *abort = 1;
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(remote(sa(&sm.abort), rank ^ 1)), "r"(1) : "memory");
  };

  if (warp == 0 && elect_one()) {
    for (size_t i = 0; i < sizeof(maps_a) / sizeof(CUtensorMap); ++i) prefetch_map(reinterpret_cast<const CUtensorMap*>(&maps_a) + i);
    for (size_t i = 0; i < sizeof(maps_b) / sizeof(CUtensorMap); ++i) prefetch_map(reinterpret_cast<const CUtensorMap*>(&maps_b) + i);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], (TA || TB) + (Cut::kCopy ? kCopyWarps : 0));
      mbar_init(&sm.empty[s], 1);
      mbar_init(&sm.landed[s], 1);
      mbar_init(&sm.fixed[s], 1);
    }
    for (int i = 0; i < kRaw * (CA + CB); ++i) {
      mbar_init(&sm.raw_full[i], 1);
      mbar_init(&sm.raw_empty[i], kCopyWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 2 * kPairOut);
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
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  JobWalk<MODE, NT, 256> walk(P, first, step);  // while the other CTA gets here
  Job j;
  bool more = walk.now(j);
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;
  uint32_t it = 0;      // stages taken
  uint32_t fixes = 0;   // a bit a stage: the parity of its next clearing

  auto blocks_of = [](const Job& q) { return (q.depth + kStepK - 1) / kStepK; };
  constexpr uint32_t kRun = Out::kRun;
  static_assert(kRun % kKB == 0, "runs of whole stages");
  // whether the last block holds rows that are not the group's (copied operands have none)
  auto to_fix = [&](const Job& q) { return MODE == kGradW && (TA || TB) && (q.depth & 15) && q.t0 + q.depth < P.m; };

  if (warp == 0) {
    // ---- loads, each CTA its halves, both counted by the first CTA's barrier ----
    uint32_t raws = 0;  // raw blocks taken
    for (; more; more = walk.next(j)) {
      const uint32_t blocks = blocks_of(j), half = (j.cols + 31) / 32 * 16;  // columns of each CTA
      const bool fix = to_fix(j);
      const int lane0 = (int)(j.lane0 + rank * 128), col0 = (int)(j.col0 + rank * half);
      const uint32_t row_a = (MODE == kGradW ? 0 : j.group * place_a.rows) + (MA ? j.t0 : (uint32_t)lane0);
      // forward: no lanes that do not exist (their results are not read)
      const bool any_a = MODE != kForward || (uint32_t)lane0 < P.lanes;
      const uint32_t bytes_a = MODE != kForward ? 2 * Smem::kHalf : P.box * 128 * (j.lane0 + 128 < P.lanes ? 2 : 1);
      if (elect_one())
        for (uint32_t kb = 0; kb < blocks; kb += kKB, ++it) {
          const uint32_t s = it % kStages, here = min((uint32_t)kKB, blocks - kb);
          if (Cut::kCopy) {
            const uint32_t q = raws % kRaw, parity = (raws / kRaw & 1) ^ 1, t = j.t0 + kb * kStepK;
            bool ok = true;
            if (CA) {
              ok = mbar_wait(&sm.raw_empty[q], parity, abort);
              if (ok) raw_load<MA>(sm.raw[q], *reinterpret_cast<const RawMaps*>(&maps_a), row_a + (MA ? kb * kStepK : 0), MA ? lane0 : (int)t, &sm.raw_full[q]);
            }
            if (CB && ok) {
              const uint32_t p = q + CA * kRaw;
              ok = mbar_wait(&sm.raw_empty[p], parity, abort);
              if (ok) raw_load<MB>(sm.raw[p], *reinterpret_cast<const RawMaps*>(&maps_b), MB ? t : (uint32_t)col0, MB ? col0 : (int)t, &sm.raw_full[p]);
            }
            if (!ok) {
              give_up();
              break;
            }
            ++raws;
          }
          if (TA || TB) {
            if (!mbar_wait(&sm.empty[s], ((it / kStages) & 1) ^ 1, abort)) {
              give_up();
              break;
            }
            const bool last = fix && kb + here == blocks;
            if (rank == 0) mbar_expect_tx(&sm.full[s], (here - last) * (TA * bytes_a + TB * 2 * Smem::kHalf));
            if (last) {
              mbar_expect_tx(&sm.landed[s], (TA + TB) * Smem::kHalf);
              fixes ^= 1u << s;
            }
            const uint32_t bar = remote(sa(&sm.full[s]), 0);
#pragma unroll
            for (uint32_t u = 0; u < kKB; ++u)
              if (u < here) {
                uint8_t* to = sm.stage[s] + 2 * u * Smem::kHalf;
                pair_load_block<MODE, TA, TB>(to, to + Smem::kHalf, reinterpret_cast<const CUtensorMap*>(&maps_a),
                                              reinterpret_cast<const CUtensorMap*>(&maps_b), j, (int)(j.t0 + (kb + u) * kStepK),
                                              lane0, col0, any_a, last && u + 1 == here ? remote(sa(&sm.landed[s]), rank) : bar);
              }
          }
        }
      if (any_of(*abort)) break;
    }
  } else if (warp == 1) {
    // ---- products, by the first CTA ----
    uint32_t n = 0, b = 0;  // accumulators taken, this one
    for (; rank == 0 && more; more = walk.next(j)) {
      const uint32_t blocks = blocks_of(j);
      const bool fix = to_fix(j);
      if (elect_one()) {
        const uint32_t idesc = idesc_f16<MODE>(P.bf16, 256, (int)((j.cols + 31) / 32 * 32));
        auto accumulator = [&]() {  // the next one, once it has been read
          b = n++ & 1;
          if (!mbar_wait_cluster(&sm.acc_empty[b], (((n - 1) >> 1) & 1) ^ 1, abort)) give_up();
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        };
        accumulator();
        for (uint32_t kb = 0; kb < blocks && !*abort; kb += kKB, ++it) {
          const uint32_t s = it % kStages, here = min((uint32_t)kKB, blocks - kb);
          const bool starts = kRun ? kb % kRun == 0 : kb == 0;
          if (kRun && starts && kb) {
            pair_commit(&sm.acc_full[b]);
            accumulator();
            if (*abort) break;
          }
          bool ok = CA || CB ? mbar_wait_cluster(&sm.full[s], (it / kStages) & 1, abort)
                             : mbar_wait(&sm.full[s], (it / kStages) & 1, abort);
          if (fix && kb + here == blocks) {
            ok = ok && mbar_wait_cluster(&sm.fixed[s], (fixes >> s) & 1, abort);
            fixes ^= 1u << s;
          }
          if (!ok) {
            give_up();
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = operand_desc<MA>(sm.stage[s]), db = operand_desc<MB>(sm.stage[s] + Smem::kHalf);
#pragma unroll
          for (uint32_t u = 0; u < kKB; ++u)
            if (u < here) {
              // grad w: no step behind the group's rows
              const uint32_t left = j.depth - (kb + u) * kStepK;
#pragma unroll
              for (uint32_t kk = 0; kk < kStepK / 16; ++kk)
                if (MODE != kGradW || kk * 16 < left)
                  mma_f16<2>(tmem + b * NT, da + u * (2 * Smem::kHalf >> 4) + kk * operand_step<MA>(),
                             db + u * (2 * Smem::kHalf >> 4) + kk * operand_step<MB>(), idesc,
                             !starts || u > 0 || kk > 0);
            }
          pair_commit(&sm.empty[s]);
        }
        pair_commit(&sm.acc_full[b]);
      }
      if (any_of(*abort)) break;
    }
  } else if (warp >= kFixer && warp < kCopier) {
    // ---- last blocks: rows behind the group's become zeros ----
    for (; more; more = walk.next(j)) {
      const uint32_t blocks = blocks_of(j), fills = (blocks + kKB - 1) / kKB;
      it += fills;
      if (!to_fix(j)) continue;
      const uint32_t s = (it - 1) % kStages;
      if (any_of(!mbar_wait(&sm.landed[s], (fixes >> s) & 1, abort))) {
        give_up();
        break;
      }
      fixes ^= 1u << s;
      const uint32_t rows = j.depth - (blocks - 1) * kStepK, to = (rows + 15) / 16 * 16;
      uint8_t* block = sm.stage[s] + (blocks - 1) % kKB * (2 * Smem::kHalf);
      for (uint32_t chunk = TA ? 0 : 2; chunk < (TB ? 4 : 2); ++chunk)
        for (uint32_t i = rows * 8 + lane; i < to * 8; i += 32)
          *reinterpret_cast<uint4*>(block + chunk * (kStepK * 128) + i * 16) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tell_written(&sm.fixed[s], block + (TA ? 0 : Smem::kHalf) + rows * 128, sm.told[kCopyGroups * kCopyWarps], rank);
    }
  } else if ((CA || CB) && warp >= kCopier) {
    // ---- copies ----
    const uint32_t mine = (warp - kCopier) / kCopyWarps, thread = (threadIdx.x - kCopier * 32) % (32 * kCopyWarps);
    uint32_t raws = 0;
    for (; more; more = walk.next(j)) {
      const uint32_t blocks = blocks_of(j), half = (j.cols + 31) / 32 * 16;
      const uint32_t lane0 = j.lane0 + rank * 128, col0 = j.col0 + rank * half;
      const uint32_t row_a = (MODE == kGradW ? 0 : j.group * place_a.rows) + (MA ? j.t0 : lane0);
      bool gone = false;
#pragma unroll 1
      for (uint32_t kb = 0; kb < blocks; ++kb, ++it, ++raws) {
        const uint32_t s = it % kStages, q = raws % kRaw, parity = raws / kRaw & 1;
        const uint32_t left = j.depth - kb * kStepK;
        if (raws % kCopyGroups != mine) continue;
        gone = !mbar_wait(&sm.empty[s], ((it / kStages) & 1) ^ 1, abort);
        if (CA && !gone) {
          gone = !mbar_wait(&sm.raw_full[q], parity, abort);
          if (!gone)
            raw_shift<MA>(thread, sm.raw[q], place_a, row_a + (MA ? kb * kStepK : 0), 128, left, sm.stage[s]);
        }
        if (CB && !gone) {
          const uint32_t p = q + CA * kRaw;
          gone = !mbar_wait(&sm.raw_full[p], parity, abort);
          if (!gone)
            raw_shift<MB>(thread, sm.raw[p], place_b, MB ? j.t0 + kb * kStepK : col0, half, left, sm.stage[s] + Smem::kHalf);
        }
        gone = any_of(gone);
        if (gone) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (CA) mbar_arrive(&sm.raw_empty[q]);
          if (CB) mbar_arrive(&sm.raw_empty[q + CA * kRaw]);
          tell_written(&sm.full[s], sm.stage[s] + (CA ? 0 : Smem::kHalf) + (thread >> 3) * 128, sm.told[warp - kCopier], rank);
        }
      }
      if (gone) give_up();
      if (any_of(*abort)) break;
    }
  } else {
    // ---- output ----
    const int quarter = warp & 3;
    const uint32_t from = (warp - 2) / 4 * kHalfTokens;
    uint32_t n = 0, b = 0;
    auto filled = [&]() {  // the next accumulator, in which a tile or a run has ended
      b = n & 1;
      const bool ok = !any_of(!mbar_wait(&sm.acc_full[b], (n >> 1) & 1, abort) || *abort);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      ++n;
      return ok;
    };
    auto read = [&]() {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_remote_relaxed(remote(sa(&sm.acc_empty[b]), 0));
    };
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
    for (; more; more = walk.next(j)) {
      const uint32_t lane0 = j.lane0 + rank * 128 + quarter * 32;
      bool ok = filled();
      if constexpr (kRun == 0) {
        if (ok) {
          out.put(P, j, mine + b * NT, lane0, from, from + kHalfTokens, sm.scratch[warp - 2]);
          read();
        }
      } else {
        float sums[kHalfTokens];
#pragma unroll
        for (int i = 0; i < kHalfTokens; ++i) sums[i] = 0.0f;
        const uint32_t runs = (blocks_of(j) + kRun - 1) / kRun;  // at least one: t is never empty here
#pragma unroll 1
        for (uint32_t r = 0; r < runs && ok; ++r) {
          if (r) ok = filled();
          if (!ok) break;
#pragma unroll
          for (int q = 0; q < kHalfTokens / 16; ++q)
            if (from + q * 16 < j.cols) {
              float f[16];
              tmem_ld16f(mine + b * NT + from + q * 16, f);
#pragma unroll
              for (int i = 0; i < 16; ++i) sums[q * 16 + i] += f[i];
            }
          read();
        }
        if (ok) out.put(P, j, sums, lane0, from);
      }
      if (!ok) {
        give_up();
        break;
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cg::this_cluster().sync();
  const bool stop = *abort;  // a wait gave up in either CTA, which told the other
  if (stop) {
    // what is still in flight ends before shared memory and TMEM are given back
    if (warp == 0 && elect_one()) {
      atomicOr(P.trap, kDeviceTimeout);
      // every stage's last use, in the first CTA for both, and each CTA's own blocks to clear
      if (TA || TB)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i) {
        if (rank == 0) mbar_wait(&sm.full[i % kStages], (i / kStages) & 1, nullptr);
      }
      if (MODE == kGradW)
        for (int s = 0; s < kStages; ++s) mbar_wait(&sm.landed[s], ((fixes >> s) & 1) ^ 1, nullptr);
      if (Cut::kCopy || MODE == kGradW) {
        const uint64_t t0 = now_ns();  // raw lines and words that tell land within microseconds, whoever waits for them
        while (now_ns() - t0 < kRawLandNs) {
        }
      }
    }
    if (warp == 1 && rank == 0 && elect_one()) {
      pair_commit(&sm.drained);
      mbar_wait(&sm.drained, 0, nullptr);
    }
  }
  __syncwarp();
  if (stop) cg::this_cluster().sync();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// ---- host --------------------------------------------------------------------------------

// Tiles of `nt` columns and `ch` lanes: at most one part-filled column tile for
// each group with rows (the offsets are on the device).
inline uint64_t product_tiles(int mode, const ProductArgs& P, uint32_t nt, uint32_t ch) {
  const uint64_t lane_tiles = (P.lanes + ch - 1) / ch;
  if (mode == kGradW) return (uint64_t)P.groups * ((P.cols + nt - 1) / nt) * lane_tiles;
  const uint64_t with_rows = P.groups < P.m ? P.groups : P.m;
  const uint64_t col_tiles = P.offsets ? P.m / nt + with_rows : (P.m + nt - 1) / nt;
  return col_tiles * lane_tiles * P.parts;
}

// Whether TMA can read rows x cols 16-bit elements at stride ld (`mats` of them at ldm).
inline bool tma_reads16(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t mats, uint64_t ldm) {
  const uint64_t lim = 1ull << 38;
  return rows && cols && aligned16(p) && (rows == 1 || (ld % 8 == 0 && ld < lim)) &&
         (mats == 1 || (ldm % 8 == 0 && ldm < lim)) && rows * (rows == 1 ? cols : ld) < lim;
}

// rows x cols elements (mats matrices of them) in boxes of 64 elements x box_rows.
inline int product_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t mats,
                       uint64_t ldm, int dims, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const uint64_t c8 = (cols + 7) & ~7ull;
  // a stride that no access uses (one row, one matrix) may be anything: any valid one stands in
  const uint64_t row = rows > 1 ? ld : c8;
  cuuint64_t dim[3] = {cols, rows, mats};
  cuuint64_t stride[2] = {2 * row, 2 * (mats > 1 ? ldm : row * rows)};
  cuuint32_t box[3] = {(cuuint32_t)kStepK, box_rows, 1}, one[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, dims, const_cast<void*>(base), dim, stride, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return 0;
}

// The two operands of a product as they lie in memory, strides in elements: A is W
// (n x k matrices, ldga apart) or, grad w, X; B is X, dY or dY.
struct Operands {
  const void* a;
  const void* b;
  uint64_t lda, ldga, ldb;
  uint64_t rows, a_cols, b_cols;  // rows and columns of one of A's matrices, columns of B
};

inline bool tma_reads_a(int mode, const ProductArgs& P, const Operands& o) {
  return tma_reads16(o.a, o.rows, o.a_cols, o.lda, mode == kGradW ? 1 : P.groups, o.ldga);
}
inline bool tma_reads_b(const ProductArgs& P, const Operands& o) { return tma_reads16(o.b, P.m, o.b_cols, o.ldb, 1, 0); }

// The maps of tiles of `lanes` and `cols`; an MN-major operand comes in boxes of 64 x 64.
inline int product_map_a(int mode, const ProductArgs& P, const Operands& o, uint32_t lanes, CUtensorMap* map) {
  return product_map(map, o.a, o.rows, o.a_cols, o.lda, mode == kGradW ? 1 : P.groups, o.ldga, mode == kGradW ? 2 : 3,
                     mode == kForward ? lanes : kStepK);
}
inline int product_map_b(int mode, const ProductArgs& P, const Operands& o, uint32_t cols, CUtensorMap* map) {
  return product_map(map, o.b, P.m, o.b_cols, o.ldb, 1, 0, 2, mode == kGradW ? kStepK : cols);
}

// The eight maps of rows x cols elements at stride ld that lie anywhere: row r by map r
// modulo 8, from its base rounded down on.
inline int raw_maps(RawMaps* maps, RawPlace* place, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, bool mn,
                    uint64_t matrix_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  for (uint64_t s = 0; s < 8; ++s) {
    const uint64_t row = s < rows ? s : 0;  // a remainder without rows is loaded all the same, and not used
    const uint64_t p = (uint64_t)(uintptr_t)base + 2 * row * ld, sh = p & 15;
    cuuint64_t dim[2] = {cols + sh / 2, s < rows ? (rows - s + 7) / 8 : 1};
    cuuint64_t stride[1] = {dim[1] > 1 ? 16 * ld : (2 * dim[0] + 15) / 16 * 16};
    cuuint32_t box[2] = {(cuuint32_t)(mn ? kLineMN : kLineK) / 2, mn ? 8u : 16u}, one[2] = {1, 1};
    const CUresult r = fn(&maps->m[s], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, (void*)(uintptr_t)(p - sh), dim, stride, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(MAPAL_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  }
  *place = {(uint32_t)((uintptr_t)base & 15), (uint32_t)(2 * ld & 15), (uint32_t)matrix_rows};
  return 0;
}

// Whether an operand that lies anywhere can be loaded raw: its matrices are one run of rows.
inline bool raw_reads(uint64_t rows, uint64_t cols, uint64_t ld, uint64_t mats, uint64_t ldm) {
  return rows && cols && ld < (1ull << 35) && (mats == 1 || ldm == rows * ld) && mats * rows < (1ull << 31);
}

template <int MODE, bool CA, bool CB, typename Out>
int launch_product_pair(const DeviceSlot& D, const Operands& o, ProductArgs P, const Out& out) {
  std::conditional_t<CA, RawMaps, CUtensorMap> ma;
  std::conditional_t<CB, RawMaps, CUtensorMap> mb;
  RawPlace pa{}, pb{};
  const uint64_t mats = MODE == kGradW ? 1 : P.groups;
  // A few lanes are loaded as the few that they are: rows behind a map's last are filled with zeros at the cost of a
  // load (the loss of 16 rows, 50257 x 2048: 65 us, where 128 rows took 58).
  P.box = P.lanes < 128 ? (P.lanes + 7) / 8 * 8 : 128;
  if constexpr (CA)
    MAPAL_TRY(raw_maps(&ma, &pa, o.a, mats * o.rows, o.a_cols, o.lda, MODE != kForward, o.rows));
  else
    MAPAL_TRY(product_map_a(MODE, P, o, P.box, &ma));
  if constexpr (CB)
    MAPAL_TRY(raw_maps(&mb, &pb, o.b, P.m, o.b_cols, o.ldb, MODE == kGradW, P.m));
  else
    MAPAL_TRY(product_map_b(MODE, P, o, 128, &mb));
  static std::atomic<uint64_t> done{0};
  auto kernel = product_pair_kernel<MODE, CA, CB, Out>;
  constexpr size_t smem = PairCut<CA, CB>::kSmem;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, smem, "product shared memory"));
  const uint64_t tiles = product_tiles(MODE, P, kPairTokens, 256), cap = D.prof.sm_count / 2;
  return launch_rows(kernel, (unsigned)((tiles < cap ? tiles : cap) * 2), pair_threads(MODE, CA, CB), smem, D.stream, 1, ma,
                     mb, pa, pb, P, out);
}

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
  uint32_t cols;   // grad w: extent of the columns' dimension (n)
  uint32_t depth;  // forward, grad x: extent of t
  uint32_t parts;  // forward, grad x: t cut into so many parts, each with its own output
  uint32_t bf16;
};

struct Job {
  uint32_t group, col0, cols, lane0;
  uint32_t t0, depth;  // the range of t
  uint32_t part;
};

// A warp's walk over the jobs of tiles of NT columns and CH lanes; every lane
// gets the answer. Lanes run fastest, so that the tiles in flight share their
// columns' operand.
template <int MODE>
struct JobWalk {
  const ProductArgs& P;
  TileWalk tiles;
  uint32_t nt, ch, lane_tiles, per_part;

  __device__ JobWalk(const ProductArgs& p, uint32_t nt_, uint32_t ch_)
      : P(p), tiles{p.offsets, p.groups, p.m, nt_, ch_, (p.lanes + ch_ - 1) / ch_, p.trap}, nt(nt_), ch(ch_) {
    lane_tiles = (p.lanes + ch_ - 1) / ch_;
    const uint32_t blocks = (p.depth + kStepK - 1) / kStepK;
    per_part = p.parts > 1 ? (blocks + p.parts - 1) / p.parts * kStepK : p.depth;
    if constexpr (MODE != kGradW) tiles.load();
  }

  __device__ bool at(uint64_t tile, Job& j) {
    if constexpr (MODE == kGradW) {
      const uint32_t col_tiles = (P.cols + nt - 1) / nt;
      const uint64_t per = (uint64_t)col_tiles * lane_tiles;
      const uint64_t g = tile / per;
      if (g >= P.groups) return false;
      const uint32_t in = (uint32_t)(tile % per);  // at most 2^32 tiles a matrix, checked on the host
      j.group = (uint32_t)g;
      j.col0 = in / lane_tiles * nt;
      j.cols = min(nt, P.cols - j.col0);
      j.lane0 = in % lane_tiles * ch;
      j.part = 0;
      uint32_t lo = 0, hi = P.m;
      if (P.offsets) {
        const int32_t a = __ldg(P.offsets + g), b = __ldg(P.offsets + g + 1);
        const bool bad = a < 0 || b < a || (uint32_t)b > P.m;
        if (bad && (threadIdx.x & 31) == 0) atomicMax(P.trap, kTrapOob);
        lo = min((uint32_t)max(a, 0), P.m);
        hi = max(lo, min((uint32_t)max(b, 0), P.m));
      }
      j.t0 = lo;
      j.depth = hi - lo;
      return true;
    } else {
      // parts run slowest: the tiles of one part share the operands' blocks
      uint32_t part = 0;
      if (P.parts > 1) {  // one group of all rows
        const uint64_t per = (uint64_t)((P.m + nt - 1) / nt) * lane_tiles;
        part = (uint32_t)(tile / per);
        tile %= per;
        if (part >= P.parts) return false;
      }
      Tile t;
      if (!tiles.at(tile, t)) return false;
      j.group = t.group;
      j.col0 = t.token0;
      j.cols = t.tokens;
      j.lane0 = t.channel0;
      j.part = part;
      j.t0 = min(part * per_part, P.depth);
      j.depth = min(per_part, P.depth - j.t0);
      return true;
    }
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

// The output as it lies in memory: column j of a job at row (grad w: row of the
// group's matrix), lanes along the row. ADD: the f32 sums so far, at the same
// places, are added first (a product taken in pieces of t).
template <int MODE, typename T, bool ADD>
struct StoreTile {
  T* out;
  const float* sums;
  uint64_t ld, ldg, ldp;  // rows, groups' matrices, parts

  // Columns [from, to) of the 32 lanes of a warp, of which this thread has `lane`.
  __device__ __forceinline__ void put(const ProductArgs& P, const Job& j, uint32_t taddr, uint32_t lane, uint32_t from,
                                      uint32_t to) const {
    const bool in = lane < P.lanes, zero = j.depth == 0;
    to = min(to, j.cols);
    const uint64_t at = (MODE == kGradW ? (uint64_t)j.group * ldg : (uint64_t)j.part * ldp) +
                        (uint64_t)(j.col0 + from) * ld + (in ? lane : 0);
    T* c = out + at;
    const float* s = ADD ? sums + at : nullptr;
    for (uint32_t j0 = from; j0 < to; j0 += 16) {
      float f[16];
      if (ADD) {
        float g[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = in && j0 + i < to ? s[i * ld] : 0.0f;
        tmem_ld16f(taddr + j0, f);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = g[i] + (zero ? 0.0f : f[i]);
        s += 16 * ld;
      } else {
        tmem_ld16f(taddr + j0, f);
        if (zero) {
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = 0.0f;
        }
      }
      if (j0 + 16 <= to) {
        if (in) {
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
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i, c += ld)
          if (in && j0 + i < to) *c = from_f32<T>(f[i]);
      }
    }
  }
};

// tiles.cuh — what the tensor-core products of rows share, in 8-bit integers and
// in 16-bit floats: the walk over the tiles of ragged groups of rows, operand
// descriptors, barriers of a pair of CTAs. Not part of the ABI.
#pragma once

#include "rows.cuh"
#include "tcgen05.cuh"

constexpr unsigned kTrapOob = 2;  // the trap flag's index_oob

constexpr int kBlockK = 128;  // bytes of k in a stage
constexpr int kHalfTokens = 128;  // that one warp writes of a tile

// Warps that write a tile of NT tokens, four (one for each quarter of the
// lanes) for every 128 tokens.
__host__ __device__ constexpr int out_warps(int nt) { return nt > kHalfTokens / 2 ? 8 : 4; }

// Shared-memory matrix descriptor, K-major, 128-byte swizzle: rows of 128
// bytes, 8-row groups `group_bytes` apart, version 1 (sm_100), layout type 2.
__device__ __forceinline__ uint64_t desc128(const void* p, uint32_t group_bytes = 1024) {
  return (uint64_t)((sa(p) & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(group_bytes >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// The address of another CTA's copy of a shared variable.
__device__ __forceinline__ uint32_t remote(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}

__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool any_of(bool p) { return __any_sync(0xffffffffu, p); }

struct Tile {
  uint32_t group, token0, tokens, channel0;
};

// A warp's walk over the tiles in ascending order; every lane gets the answer.
struct TileWalk {
  const int32_t* offsets;
  uint32_t groups, m, nt, channels, channel_tiles;
  unsigned* trap;
  uint32_t base = 0, before = 0;      // the chunk's first group, token tiles before it
  uint32_t lo = 0, hi = 0, incl = 0;  // this lane's group: rows, token tiles up to and with it
  uint32_t chunk = 0;                 // token tiles of the chunk
  uint32_t least = 0;                 // once an offset was bad: the largest so far
  bool broken = false;

  __device__ void load() {
    const uint32_t lane = threadIdx.x & 31, g = base + lane;
    lo = hi = 0;
    bool bad = false;
    if (g < groups) {
      if (offsets) {
        const int32_t a = __ldg(offsets + g), b = __ldg(offsets + g + 1);
        bad = a < 0 || b < a || (uint32_t)b > m;
        lo = (uint32_t)max(a, 0);
        hi = (uint32_t)max(b, 0);
      } else {
        hi = m;
      }
    }
    broken = __any_sync(0xffffffffu, bad || broken);
    if (broken) raise(bad);
    incl = (hi - lo + nt - 1) / nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    chunk = __shfl_sync(0xffffffffu, incl, 31);
  }

  // Bad offsets: each becomes the largest up to it, at most m, so that groups
  // still do not share rows and there are no more tiles than rows allow.
  __device__ __forceinline__ void raise(bool bad) {
    const uint32_t lane = threadIdx.x & 31;
    if (bad) atomicMax(trap, kTrapOob);
    lo = min(lo, m);
    hi = max(lo, min(hi, m));
    uint32_t top = hi;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, top, o);
      if (lane >= o) top = max(top, up);
    }
    const uint32_t below = __shfl_up_sync(0xffffffffu, top, 1);
    lo = max(lo, max(least, lane ? below : 0u));
    hi = max(lo, hi);
    least = max(least, __shfl_sync(0xffffffffu, top, 31));
  }

  __device__ bool at(uint64_t tile, Tile& t) {
    t.channel0 = (uint32_t)(tile % channel_tiles) * channels;
    return find(tile / channel_tiles, t);
  }

  // The group and tokens of a token tile.
  __device__ __forceinline__ bool find(uint64_t token_tile, Tile& t) {
    while (token_tile >= (uint64_t)before + chunk) {
      base += 32;
      if (base >= groups) return false;
      before += chunk;
      load();
    }
    const uint32_t want = (uint32_t)(token_tile - before);
    const int src = __ffs(__ballot_sync(0xffffffffu, incl > want)) - 1;
    const uint32_t glo = __shfl_sync(0xffffffffu, lo, src), ghi = __shfl_sync(0xffffffffu, hi, src);
    const uint32_t first = __shfl_sync(0xffffffffu, incl, src) - (ghi - glo + nt - 1) / nt;
    t.group = base + src;
    t.token0 = glo + (want - first) * nt;
    t.tokens = min(nt, ghi - t.token0);
    return true;
  }
};

__device__ __forceinline__ void pair_commit(uint64_t* bar) {  // in both CTAs
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(sa(bar)),
      "h"((uint16_t)3)
      : "memory");
}


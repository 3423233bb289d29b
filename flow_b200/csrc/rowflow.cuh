// rowflow.cuh — how the row-wise kernels for many rows move through memory:
// groups of threads that share rows, and a ring that brings rows in ahead.
// Not part of the ABI.
#pragma once

#include "rows.cuh"

// Threads of a block that share a row: 8 or 16 lanes of a warp (SUB), a warp,
// which need no barrier, or several warps, which meet at a named barrier of
// their own.
template <bool SUB>
struct Group {
  int size, tid, id;
  __device__ explicit Group(int g) : size(g), tid(threadIdx.x % g), id(threadIdx.x / g) {}
  __device__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(size) : "memory"); }
  // N sums over the group at once, in every thread. Lanes halve the values
  // they carry while they add, so 4 sums take 6 shuffles instead of 20. `red`
  // is the group's own, and not that of the sums before (two sets taken in
  // turn are enough).
  template <int N>
  __device__ void sums(float (&a)[N], float (*red)[16]) const {
    static_assert(N == 1 || N == 2 || N == 4, "");
    if constexpr (SUB) {  // other groups of the warp may have no row left
      const unsigned lanes = ((1u << size) - 1) << (threadIdx.x & 31 & ~(size - 1));
#pragma unroll
      for (int k = 0; k < N; ++k)
        for (int o = size / 2; o > 0; o >>= 1) a[k] += __shfl_xor_sync(lanes, a[k], o);
      return;
    }
    constexpr unsigned kAll = 0xffffffffu;
    constexpr int L = 32 / N;  // lanes that end with the same value
    const int lane = tid & 31;
    float v;
    if constexpr (N == 1) {
      v = a[0];
    } else if constexpr (N == 2) {
      const bool up = lane & 16;
      v = (up ? a[1] : a[0]) + __shfl_xor_sync(kAll, up ? a[0] : a[1], 16);
    } else {
      const bool up = lane & 16, up2 = lane & 8;
      const float p = (up ? a[2] : a[0]) + __shfl_xor_sync(kAll, up ? a[0] : a[2], 16);
      const float q = (up ? a[3] : a[1]) + __shfl_xor_sync(kAll, up ? a[1] : a[3], 16);
      v = (up2 ? q : p) + __shfl_xor_sync(kAll, up2 ? p : q, 8);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    if (size > 32) {
      const int at = lane % L, warps = size / 32;
      if (at == 0) red[lane / L][tid >> 5] = v;
      sync();
      v = at < warps ? red[lane / L][at] : 0.0f;
      if (L < 16 && at + L < warps) v += red[lane / L][at + L];
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) a[k] = __shfl_sync(kAll, v, k * L);
  }
  __device__ float sum(float a, float* red) const {
    a = warp_sum(a);
    if (size == 32) return a;
    const int lane = tid & 31, warp = tid >> 5;
    if (lane == 0) red[warp] = a;
    sync();
    return warp_sum(lane < size / 32 ? red[lane] : 0.0f);
  }
};
constexpr int kMostGroups = 8;  // of more than a warp in a block

// Rows arrive through a ring in shared memory: every thread copies its own
// elements with cp.async and reads them back itself, so there is nothing to
// wait for but its own copies, and rows stay in flight without holding
// registers. 16-bit rows at odd addresses, which cp.async cannot copy, are
// loaded into registers one turn ahead.

constexpr int kFlow = 512;  // threads of a block; one block an SM

// V: elements of an access; ARRAYS: 1 (x) or 2 (x and dy).
template <typename T, int V, int EACH, int ROWS, int ARRAYS>
struct Ring {
  using P = Pack<T, V>;
  static constexpr int NV = EACH / V;
  static constexpr bool kAsync = sizeof(P) >= 4;
  static constexpr int kSlots = ARRAYS * ROWS * NV;  // of a thread in a stage
  static constexpr int kStages = !kAsync ? 1 : sizeof(T) == 4 ? 3 : 4;
  static constexpr size_t kBytes = kAsync ? (size_t)kStages * kSlots * sizeof(P) * kFlow : 0;
  P* base;
  P ahead[kAsync ? 1 : kSlots];
  int stage = 0;
  __device__ explicit Ring(void* p) : base(static_cast<P*>(p)) {}

  __device__ __forceinline__ P* slot(int st, int s) { return base + (size_t)(st * kSlots + s) * kFlow + threadIdx.x; }
  __device__ __forceinline__ void copy(int st, int s, const T* from) {
    if constexpr (kAsync) {
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot(st, s));
      if constexpr (sizeof(P) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
    } else {
      ahead[s] = ld_once(reinterpret_cast<const P*>(from));
    }
  }
  __device__ __forceinline__ void commit() {
    if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // This turn's rows are there.
  __device__ __forceinline__ void wait() {
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
  }
  __device__ __forceinline__ P take(int s) { return kAsync ? *slot(stage, s) : ahead[kAsync ? 0 : s]; }
  __device__ __forceinline__ void next() { stage = stage + 1 == kStages ? 0 : stage + 1; }
};

// How the kernels for many rows are launched: threads of a group, of a block,
// blocks.
struct Plan {
  int group, threads;
  unsigned blocks;
};

inline Plan flow_plan(uint64_t rows, uint64_t d, int sms, uint64_t each, uint64_t turn) {
  Plan p;
  p.group = d <= 64 ? 8 : d <= 128 ? 16 : (int)((d + 32 * each - 1) / (32 * each)) * 32;
  p.threads = kFlow / p.group * p.group;
  const uint64_t groups = p.threads / p.group, want = (rows + groups * turn - 1) / (groups * turn);
  p.blocks = (unsigned)(want < (uint64_t)sms ? want : sms);
  return p;
}

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
  template <typename G>
  __device__ Ring(void* p, const G&) : base(static_cast<P*>(p)) {}

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
  __device__ __forceinline__ void next_stage() { stage = stage + 1 == kStages ? 0 : stage + 1; }
};

// ---- rows that begin or end inside an access ------------------------------------
//
// Rows whose starts or lengths are no multiple of 16 bytes still move in whole
// 16-byte accesses: a thread's columns are those of an aligned access of the
// output, whose first and last access in a row are in part another row's and
// are written element by element. An input whose rows begin elsewhere within
// their 16 bytes is shifted into place on the way out of the ring, from a
// thread's own aligned word and the next thread's. Where a row begins goes
// round with the rows, so a unit (a group, or a warp of several) takes rows of
// one class modulo `period`, which begin alike: its columns, weights and sums
// over rows stay as they are. What is left is instructions and their latencies:
// at 60000 x 1021 the 15 warps of an SM fill 55 (forward) and 57 % (gradient) of
// the issue slots and wait for results of their own and at the sums' barriers,
// with HBM at 24 and 37 % of its peak; rows to 8 bits, 16384 x 8191: 9 warps,
// 46 % and 43 %. Layer norm and its
// gradient, bf16: 60000 x 1021 93 and 112 us, element by element 104 and 182;
// 30000 x 2047 77 and 138, 109 and 188; 12000 x 5001 83 and 165, 169 and 794.
// Rows to 8 bits: 16384 x 8191 101 us, with shifted words 133, one by one 187.
//
// EDGE 0: rows are whole accesses; 1: an input's rows begin as the output's do
// within their 16 bytes; 2: they may begin elsewhere.

// Elements a thread of the device from which on rows at odd places take those
// kernels too (1300 x 1021 f16: 5.2 us, one by one 7.1; 100 x 1001 4.0 both).
constexpr uint64_t kEdgeTurns = 16;

// Values that are worth a register: made again where they are used, as the
// compiler prefers, they cost a third of the instructions (10 to 25% of the time).
__device__ __forceinline__ void pin(uint32_t& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void pin(int& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void pin(uint64_t& v) { asm volatile("" : "+l"(v)); }
template <typename T>
__device__ __forceinline__ void pin(T*& v) {
  asm volatile("" : "+l"(v));
}

template <bool SUB, int EDGE, int ROWS>
struct Turns {
  uint64_t first, step, rows;  // counted in rows of the class
  uint32_t cls = 0, period = 1;
  __device__ Turns(const Group<SUB>& G, uint32_t p, uint64_t all_rows) : rows(all_rows) {
    const uint32_t groups = blockDim.x / G.size, id = blockIdx.x * groups + G.id, all = gridDim.x * groups;
    if constexpr (!EDGE) {
      first = (uint64_t)id * ROWS;
      step = (uint64_t)all * ROWS;
    } else {
      const uint32_t per = SUB ? 32 / G.size : 1, unit = id / per;
      cls = unit % p;
      period = p;
      first = ((uint64_t)(unit / p) * per + id % per) * ROWS;
      step = (uint64_t)(all / per / p) * per * ROWS;
      rows = all_rows > cls ? (all_rows - cls + p - 1) / p : 0;
    }
  }
  // Elements between a 16-byte boundary and the class's rows (arrays begin at one).
  template <typename T>
  __device__ __forceinline__ int shift(uint64_t ld) const {
    return EDGE ? (int)(cls * ld % (16 / sizeof(T))) : 0;
  }
  // Row stride and first row of the class, from the array's.
  __device__ __forceinline__ uint64_t stride(uint64_t ld) const { return EDGE ? ld * period : ld; }
  template <typename T>
  __device__ __forceinline__ T* at(T* p, uint64_t ld) const {
    return EDGE && p ? p + cls * ld : p;
  }
};

// Which elements of a thread's columns are its row's, V bits for each access.
template <int V, int NV>
struct Mine {
  static_assert(V * NV <= 32, "");
  static constexpr uint32_t kAll = (1u << V) - 1;
  uint32_t bits = 0;
  __device__ Mine(int group, int tid, int from, int to) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = (j * group + tid) * V + e;
        bits |= (i >= from && i < to ? 1u : 0u) << (j * V + e);
      }
    pin(bits);
  }
  __device__ __forceinline__ uint32_t at(int j) const { return (bits >> (j * V)) & kAll; }
};

// For whole rows: nothing to know.
struct Whole {
  static constexpr int back = 0, by = 0;
  template <typename... A>
  __device__ explicit Whole(const A&...) {}
};

// Zeros for what is not the row's: one access's masks stay in registers, those
// of several are made again where they are needed.
template <typename P, int V, int NV>
struct Masks {
  uint32_t w[4];
  const Mine<V, NV>& part;
  __device__ explicit Masks(const Mine<V, NV>& p) : part(p) {
    P ones;
#pragma unroll
    for (int i = 0; i < P::W; ++i) ones.w[i] = 0xffffffffu;
    ones.keep(p.at(0));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = ones.w[i % P::W];
      if constexpr (NV == 1) pin(w[i]);
    }
  }
  __device__ __forceinline__ void operator()(P& p, int j) const {
    if constexpr (NV == 1) {
#pragma unroll
      for (int i = 0; i < P::W; ++i) p.w[i] &= w[i];
    } else if (part.at(j) != part.kAll) {
      p.keep(part.at(j));
    }
  }
};

// The ring for such rows. A warp's words lie side by side, with room for the
// word behind those of each of its groups.
template <typename T, int EACH, int ROWS, int ARRAYS, bool SUB, bool SHIFTED>
struct EdgeRing {
  static constexpr int V = 16 / sizeof(T), NV = EACH / V;
  using P = Pack<T, V>;
  static constexpr int kSlots = ARRAYS * ROWS * NV;
  static constexpr int kStages = sizeof(T) == 4 ? 3 : 4;
  static constexpr int kWords = SUB ? 36 : 33;  // of a warp in a slot
  static constexpr size_t kBytes = (size_t)kStages * kSlots * (kFlow / 32) * kWords * 16;
  P *own, *next;
  uint32_t lanes;  // that read each other's words
  bool last;
  int stage = 0;
  __device__ EdgeRing(void* p, const Group<SUB>& G) {
    const int lane = threadIdx.x & 31, size = SUB ? G.size : 32;
    lanes = SUB ? ((1u << size) - 1) << (lane & ~(size - 1)) : 0xffffffffu;
    last = (lane & (size - 1)) == size - 1;
    own = static_cast<P*>(p) + (threadIdx.x / 32) * kWords + lane;
    next = last ? own - lane + 32 + lane / size : own + 1;
  }
  static __device__ __forceinline__ size_t slot(int st, int s) { return (size_t)(st * kSlots + s) * (kFlow / 32) * kWords; }
  static __device__ __forceinline__ void copy(P* to, const T* from, int n) {  // n elements, zeros behind them
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
                 "r"(min(n, V) * (int)sizeof(T))
                 : "memory");
  }
  // A thread's word of a row, of which `left` elements are the row's, and where
  // words are shifted the one behind the last thread's.
  __device__ __forceinline__ void bring(int st, int s, const T* from, int left) {
    if (left > 0) copy(own + slot(st, s), from, left);
    if (SHIFTED && last && left > V) copy(next + slot(st, s), from + V, left - V);
  }
  __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // This turn's rows are there, for the threads that share them.
  __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    if constexpr (SHIFTED) __syncwarp(lanes);
  }
  // An access of the output's columns, `by` elements into the words.
  __device__ __forceinline__ P take(int s, int by) const {
    const P* a = own + slot(stage, s);
    if constexpr (!SHIFTED) return *a;
    P p;
    const uint4 v = straddle(*reinterpret_cast<const uint4*>(a), *reinterpret_cast<const uint4*>(next + slot(stage, s)),
                             (uint32_t)by * sizeof(T));
    p.w[0] = v.x, p.w[1] = v.y, p.w[2] = v.z, p.w[3] = v.w;
    return p;
  }
  // The words may be overwritten.
  __device__ __forceinline__ void taken() const {
    if constexpr (SHIFTED) __syncwarp(lanes);
  }
  __device__ __forceinline__ void next_stage() { stage = stage + 1 == kStages ? 0 : stage + 1; }
};

// An input's words against the output's accesses: a thread's word `back`
// accesses before its own, `by` elements of which come before its columns.
template <int V, int NV>
struct Input {
  int back, by, left[NV];
  __device__ Input(int group, int tid, int d, int in, int out) : back(in < out), by(in < out ? in - out + V : in - out) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int word = j * group + tid - back;
      left[j] = word < 0 ? 0 : d + in - word * V;
      pin(left[j]);
    }
  }
};

// Classes of rows by where they begin, for accesses of v elements (a power of
// two) and these row strides.
inline uint32_t edge_period(uint64_t rows, std::initializer_list<uint64_t> lds, uint32_t v) {
  uint32_t p = 1;
  if (rows > 1)
    for (const uint64_t ld : lds)
      while (ld * p % v) p *= 2;
  return p;
}

// How the kernels for many rows are launched: threads of a group, of a block,
// blocks.
struct Plan {
  int group, threads;
  unsigned blocks;
};

// Rows that a block has at once.
inline uint64_t rows_at_once(uint64_t span, uint64_t each, uint64_t turn) {
  return kFlow / ((span + 32 * each - 1) / (32 * each) * 32) * turn;
}

// d: columns that a group spans. The number of units is a multiple of period.
template <bool LANES = true>  // groups of less than a warp
inline Plan flow_plan(uint64_t rows, uint64_t d, int sms, uint64_t each, uint64_t turn, uint32_t period = 1) {
  Plan p;
  p.group = LANES && d <= 64 ? 8 : LANES && d <= 128 ? 16 : (int)((d + 32 * each - 1) / (32 * each)) * 32;
  p.threads = kFlow / p.group * p.group;
  const uint64_t groups = p.threads / p.group, want = (rows + groups * turn - 1) / (groups * turn);
  p.blocks = (unsigned)(want < (uint64_t)sms ? want : sms);
  const unsigned units = p.group < 32 ? p.threads / 32 : (unsigned)groups;
  unsigned more = p.blocks;
  while (more * units % period) ++more;
  if (more <= (unsigned)sms) p.blocks = more;
  while (p.blocks * units % period) --p.blocks;
  return p;
}

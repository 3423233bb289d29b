// dropout.cu — dropout with a mask that is never stored, added to a residual
// (mapal_gpu_dropout). No counterpart in the reference.
//
// Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011) turns a counter into 128 random bits by ten rounds of two
// 32 x 32 -> 64 bit products: 16 bits for each of 8 elements of a row. The counter is
// made of the place (row, column), so any order of the elements, any stride and
// the gradient's call give the same mask.
#include <cmath>

#include "rows.cuh"

namespace {

constexpr int kThreads = 256;

struct Key {
  uint32_t k[10][2];  // of each round
  uint32_t c2, c3;
};

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, const Key& k) {
  uint32_t c2 = k.c2, c3 = k.c3;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k.k[i][0];
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k.k[i][1];
    c3 = (uint32_t)p0;
  }
  return make_uint4(c0, c1, c2, c3);
}

struct DropArgs {
  const void* x;
  const void* residual;
  void* y;
  const unsigned long long* rng;
  uint64_t ldx, ldr, ldy, rows;
  uint32_t d, blocks;  // elements of a row, and eights of them
  uint32_t lanes;      // threads on a row, a power of two
  uint32_t limit;      // in both halves of a word; p = 1 does not get this far
  float scale;
};

__device__ __forceinline__ Key key_of(const DropArgs& A) {
  const unsigned long long key = __ldg(A.rng), place = __ldg(A.rng + 1);
  Key k;
  k.c2 = (uint32_t)place, k.c3 = (uint32_t)(place >> 32);
#pragma unroll
  for (uint32_t i = 0; i < 10; ++i) {
    k.k[i][0] = (uint32_t)key + i * 0x9E3779B9u;
    k.k[i][1] = (uint32_t)(key >> 32) + i * 0xBB67AE85u;
  }
  return k;
}

// Which of the eight elements are kept: two 16-bit comparisons an instruction.
__device__ __forceinline__ void keeps(const uint4& w, uint32_t limit2, bool (&k)[8]) {
  __vibmax_u16x2(w.x, limit2, &k[1], &k[0]);
  __vibmax_u16x2(w.y, limit2, &k[3], &k[2]);
  __vibmax_u16x2(w.z, limit2, &k[5], &k[4]);
  __vibmax_u16x2(w.w, limit2, &k[7], &k[6]);
}

template <typename T>
__device__ __forceinline__ void drop_one(const DropArgs& A, const T* x, const T* res, T* y, bool keep) {
  const float g = res ? to_f32(*res) : 0.0f;
  *y = from_f32<T>(keep ? __fmaf_rn(to_f32(*x), A.scale, g) : g);
}

// Rows on 16-byte boundaries. Bound by HBM: a thread takes kAhead eights of a row, all
// of their loads before the first bits, so that the generator's 10 rounds (40 multiply-and-xor
// instructions) run while they are under way. A row's last part eight goes
// element by element.
constexpr int kAhead = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropArgs A) {
  constexpr int V = 16 / sizeof(T), N = 8 / V;  // elements of an access, accesses of an eight
  using P = Pack<T, V>;
  const uint32_t in_row = threadIdx.x & (A.lanes - 1), per_block = kThreads / A.lanes;
  grid_wait();
  grid_go();
  const Key k = key_of(A);
  const T* x = static_cast<const T*>(A.x);
  const T* res = static_cast<const T*>(A.residual);
  T* y = static_cast<T*>(A.y);
  const uint32_t whole = A.d / 8, wide = A.lanes * kAhead;  // eights that a row's threads take at a time
  const uint32_t row_in = threadIdx.x / A.lanes;
  auto take = [&](uint64_t r, uint32_t b0) {
    const T *xr = x + r * A.ldx, *rr = res ? res + r * A.ldr : nullptr;
    T* yr = y + r * A.ldy;
    P xv[kAhead][N], rv[kAhead][N];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t b = b0 + u * A.lanes;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (b < whole) {
          xv[u][i] = ld_once(reinterpret_cast<const P*>(xr + b * 8ull + i * V));
          if (res) rv[u][i] = ld_once(reinterpret_cast<const P*>(rr + b * 8ull + i * V));
        }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t b = b0 + u * A.lanes;
      if (b >= A.blocks) return;
      bool keep[8];
      keeps(philox(b, (uint32_t)r, k), A.limit, keep);
      if (b < whole) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float f[V], g[V] = {};
          xv[u][i].get(f);
          if (res) rv[u][i].get(g);
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] = keep[i * V + e] ? __fmaf_rn(f[e], A.scale, g[e]) : g[e];
          P o;
          o.set(f);
          st_once(reinterpret_cast<P*>(yr + b * 8ull + i * V), o);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (b * 8 + e < A.d)
            drop_one(A, xr + b * 8ull + e, rr ? rr + b * 8ull + e : nullptr, yr + b * 8ull + e, keep[e]);
      }
    }
  };
  for (uint64_t r = blockIdx.x * (uint64_t)per_block + row_in; r < A.rows; r += (uint64_t)gridDim.x * per_block)
    for (uint64_t first = (uint64_t)blockIdx.y * wide; first < A.blocks; first += (uint64_t)gridDim.y * wide)
      take(r, (uint32_t)first + in_row);
}

// Rows anywhere: a warp takes 256 elements, an eight's bits a thread, and gives them out
// by shuffles, so that neighbouring threads access neighbouring elements (V of them; eight
// in a row by each thread took 36 us for 5003 x 1021 f16 with gradient).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) dropout_loose_kernel(const DropArgs A) {
  using P = Pack<T, V>;
  constexpr int kTurns = 8 / V;
  const uint32_t lane = threadIdx.x & 31;
  grid_wait();
  grid_go();
  const Key k = key_of(A);
  const T* x = static_cast<const T*>(A.x);
  const T* res = static_cast<const T*>(A.residual);
  T* y = static_cast<T*>(A.y);
  const uint32_t pieces = (A.blocks + 31) / 32;
  const uint64_t items = A.rows * pieces, step = (uint64_t)gridDim.x * (kThreads / 32);
  for (uint64_t item = (uint64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; item < items; item += step) {
    const uint64_t r = item >> 32 ? item / pieces : (uint32_t)item / pieces;  // the 64-bit division takes 100 instructions
    const uint32_t b0 = (uint32_t)(item - r * pieces) * 32;
    const uint64_t e0 = b0 * 8ull + lane * V;
    const T *xr = x + r * A.ldx + e0, *rr = res ? res + r * A.ldr + e0 : nullptr;
    T* yr = y + r * A.ldy + e0;
    const uint32_t left = A.d > e0 ? (uint32_t)min((uint64_t)A.d - e0, (uint64_t)0xffffffffu) : 0;
    P xv[kTurns], rv[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      if (i * 32 * V < left) {
        xv[i] = *reinterpret_cast<const P*>(xr + i * 32 * V);
        if (res) rv[i] = *reinterpret_cast<const P*>(rr + i * 32 * V);
      }
    bool keep[8];
    keeps(philox(b0 + lane, (uint32_t)r, k), A.limit, keep);
    uint32_t m = 0;  // which of this thread's eight are kept
#pragma unroll
    for (int c = 0; c < 8; ++c) m |= keep[c] ? 1u << c : 0u;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const uint32_t e = i * 32 * V + lane * V;  // of the warp's 256
      const uint32_t bits = __shfl_sync(0xffffffffu, m, e / 8) >> (e & 7);
      if (i * 32 * V < left) {
        float f[V], g[V] = {};
        xv[i].get(f);
        if (res) rv[i].get(g);
#pragma unroll
        for (int c = 0; c < V; ++c) f[c] = bits & (1u << c) ? __fmaf_rn(f[c], A.scale, g[c]) : g[c];
        P o;
        o.set(f);
        *reinterpret_cast<P*>(yr + i * 32 * V) = o;
      }
    }
  }
}

template <typename T>
int launch(const DeviceSlot& D, DropArgs A) {
  // a row's threads: enough for its eights, kAhead each
  for (A.lanes = 1; A.lanes * kAhead < A.blocks && A.lanes < kThreads;) A.lanes *= 2;
  const uint64_t per_block = kThreads / A.lanes, pieces = (A.blocks + A.lanes * kAhead - 1) / (A.lanes * kAhead);
  // 16 bits: few blocks that walk the rows, so that the key's schedule is made once for many eights (16384 x 8192 bf16
  // with residual 147 us with a block an item, 125 with these). f32 is bound by HBM (8000 x 8192
  // with residual 115 us, 78 without), and becomes 126 us with them.
  const uint64_t groups = (A.rows + per_block - 1) / per_block, y = pieces < 64 ? pieces : 64;
  const uint64_t most = sizeof(T) == 2 ? (8ull * D.prof.sm_count + y - 1) / y : 1u << 20;
  const dim3 grid((unsigned)(groups < most ? groups : most), (unsigned)y);
  return launch_rows(dropout_kernel<T>, grid, kThreads, 0, D.stream, 1, A);
}

template <typename T, int V>
int launch_loose(const DeviceSlot& D, const DropArgs& A) {
  const uint64_t items = A.rows * ((A.blocks + 31) / 32), blocks = (items + kThreads / 32 - 1) / (kThreads / 32), most = 1u << 20;
  return launch_rows(dropout_loose_kernel<T, V>, (unsigned)(blocks < most ? blocks : most), kThreads, 0, D.stream, 1, A);
}

}  // namespace

extern "C" int mapal_gpu_dropout(MapalGpuCtx* ctx, const MapalDropoutSite* site, const void* x, const void* residual,
                                 const uint64_t* rng, void* y) {
  return guarded([&]() -> int {
    if (!site) return set_error(MAPAL_ERR_INVALID, "site is null");
    const MapalDropoutSite& s = *site;
    const int es = dtype_bytes(s.dtype);
    if (es < 2) return set_error(MAPAL_ERR_INVALID, "rows are f32, f16 or bf16");
    if (!(s.p >= 0.0 && s.p <= 1.0)) return set_error(MAPAL_ERR_INVALID, "p is not between 0 and 1");
    if (s.rows > 0x7fffffffull || s.d > 0x7fffffffull) return set_error(MAPAL_ERR_UNSUPPORTED, "2^31 rows or elements of a row, or more");
    if (!rows_ok(s.rows, s.d, s.ldx, es) || !rows_ok(s.rows, s.d, s.ldy, es) ||
        (residual && !rows_ok(s.rows, s.d, s.ldr, es)))
      return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
    if (s.rows == 0 || s.d == 0) return 0;
    if (!x || !y || !rng) return set_error(MAPAL_ERR_INVALID, "null x, y or rng");
    if (((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) & (es - 1) || (uintptr_t)rng & 7)
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    if (s.rows > 1 && ((y == x && s.ldy != s.ldx) || (y == residual && s.ldy != s.ldr)))
      return set_error(MAPAL_ERR_INVALID, "y is x or residual, but not at the same stride");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    DropArgs A{};
    A.x = x;
    A.residual = residual;
    A.y = y;
    A.rng = reinterpret_cast<const unsigned long long*>(rng);
    A.ldx = s.ldx;
    A.ldr = s.ldr;
    A.ldy = s.ldy;
    A.rows = s.rows;
    A.d = (uint32_t)s.d;
    A.blocks = (uint32_t)((s.d + 7) / 8);
    const uint32_t limit = (uint32_t)std::lrint(s.p * 65536.0);
    if (limit == 65536) {  // nothing of x is left
      if (residual != y) MAPAL_TRY(copy_rows(y, s.ldy * es, residual, s.ldr * es, s.d * es, s.rows, D.stream));
      return finish(ctx, 0, false);
    }
    A.limit = limit * 0x10001u;
    A.scale = (float)(65536.0 / (65536 - limit));
    int width = align_of(x, s.ldx * es, s.rows);
    for (const int o : {align_of(y, s.ldy * es, s.rows), residual ? align_of(residual, s.ldr * es, s.rows) : 16})
      width = o < width ? o : width;
    auto half = [&](auto t) {
      using T = decltype(t);
      if (width >= 16) return launch<T>(D, A);
      if (width >= 4 && s.d % 2 == 0) return launch_loose<T, 2>(D, A);
      return launch_loose<T, 1>(D, A);
    };
    MAPAL_TRY(s.dtype == MAPAL_DTYPE_F32 ? (width >= 16 ? launch<float>(D, A) : launch_loose<float, 1>(D, A))
              : s.dtype == MAPAL_DTYPE_F16 ? half(__half{})
                                           : half(__nv_bfloat16{}));
    return finish(ctx, 0, false);
  });
}

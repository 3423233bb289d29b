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
  uint32_t k0, k1, c2, c3;
};

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, const Key& k) {
  uint32_t c2 = k.c2, c3 = k.c3, k0 = k.k0, k1 = k.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
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
  uint32_t limit;
  float scale;
};

// A thread takes eights of a row, `lanes` threads of a block a row, V elements an access.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropArgs A) {
  using P = Pack<T, V>;
  constexpr int N = 8 / V;  // accesses
  const uint32_t in_row = threadIdx.x & (A.lanes - 1), per_block = kThreads / A.lanes;
  grid_wait();
  grid_go();
  const unsigned long long key = __ldg(A.rng), place = __ldg(A.rng + 1);
  const Key k{(uint32_t)key, (uint32_t)(key >> 32), (uint32_t)place, (uint32_t)(place >> 32)};
  const T* x = static_cast<const T*>(A.x);
  const T* res = static_cast<const T*>(A.residual);
  T* y = static_cast<T*>(A.y);
  const uint32_t pieces = (A.blocks + A.lanes - 1) / A.lanes;
  const uint64_t row_groups = (A.rows + per_block - 1) / per_block, items = row_groups * pieces;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint64_t r = item / pieces * per_block + threadIdx.x / A.lanes;
    const uint32_t b = (uint32_t)(item % pieces) * A.lanes + in_row;
    if (r >= A.rows || b >= A.blocks) continue;
    const uint32_t n = min(8u, A.d - b * 8);
    const uint64_t at = (uint64_t)b * 8;
    P xv[N], rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * V < n) xv[i] = *reinterpret_cast<const P*>(x + r * A.ldx + at + i * V);
      if (res && i * V < n) rv[i] = *reinterpret_cast<const P*>(res + r * A.ldr + at + i * V);
    }
    const uint4 w = philox(b, (uint32_t)r, k);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * V < n) {
        float f[V], g[V];
        xv[i].get(f);
        if (res)
          rv[i].get(g);
        else
#pragma unroll
          for (int e = 0; e < V; ++e) g[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = i * V + e;
          const uint32_t bits = c & 1 ? words[c / 2] >> 16 : words[c / 2] & 0xffffu;
          f[e] = bits >= A.limit ? __fmaf_rn(f[e], A.scale, g[e]) : g[e];
        }
        P o;
        o.set(f);
        *reinterpret_cast<P*>(y + r * A.ldy + at + i * V) = o;
      }
  }
}

template <typename T, int V>
int launch(const DeviceSlot& D, const DropArgs& A) {
  const uint64_t per_block = kThreads / A.lanes, pieces = (A.blocks + A.lanes - 1) / A.lanes;
  const uint64_t items = (A.rows + per_block - 1) / per_block * pieces, cap = 32ull * D.prof.sm_count;
  return launch_rows(dropout_kernel<T, V>, (unsigned)(items < cap ? items : cap), kThreads, 0, D.stream, 1, A);
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
    for (A.lanes = 1; A.lanes < A.blocks && A.lanes < kThreads;) A.lanes *= 2;
    A.limit = (uint32_t)std::lrint(s.p * 65536.0);
    A.scale = A.limit < 65536 ? (float)(65536.0 / (65536 - A.limit)) : 0.0f;
    int width = align_of(x, s.ldx * es, s.rows);
    for (const int o : {align_of(y, s.ldy * es, s.rows), residual ? align_of(residual, s.ldr * es, s.rows) : 16,
                        align_of(nullptr, s.d * es, 2)})
      width = o < width ? o : width;
    auto half = [&](auto t) {
      using T = decltype(t);
      if (width >= 16) return launch<T, 8>(D, A);
      if (width >= 4) return launch<T, 2>(D, A);
      return launch<T, 1>(D, A);
    };
    MAPAL_TRY(s.dtype == MAPAL_DTYPE_F32 ? (width >= 16 ? launch<float, 4>(D, A) : launch<float, 1>(D, A))
              : s.dtype == MAPAL_DTYPE_F16 ? half(__half{})
                                           : half(__nv_bfloat16{}));
    return finish(ctx, 0, false);
  });
}

// matmul_i8.cu — products in 8-bit integers with a scale for each row of A and
// each row (output channel) of B, for one matrix or one per group of rows
// (mapal_gpu_matmul_i8). No counterpart in the reference.
//
// C[i, j] = (sum_k A[i, k]*B[g][j, k]) * scale_a[i] * scale_b[g][j]. The sum
// is exact in 32 bits for k < 2^17 (127^2 and even 128^2 times k stays below
// 2^31), so any split or order of it gives the same bits; the float steps are
// one conversion and two multiplications, each rounded to f32.
#include "rows.cuh"

namespace {

constexpr unsigned kTrapOob = 2;  // the trap flag's index_oob

template <typename T>
__device__ __forceinline__ T scaled(int acc, float sa, float sb) {
  return from_f32<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc), sa), sb));
}

// Group g's rows [lo, hi), clamped to [0, m] and ascending; raises the trap
// where the offsets are not.
__device__ __forceinline__ void group_rows(const int32_t* offsets, uint32_t g, uint32_t m, unsigned* trap, uint32_t& lo,
                                           uint32_t& hi) {
  const int32_t a = __ldg(offsets + g), b = __ldg(offsets + g + 1);
  if (a < 0 || b < a || (uint32_t)b > m) atomicMax(trap, kTrapOob);
  lo = a < 0 ? 0u : min((uint32_t)a, m);
  hi = b < 0 ? lo : max(lo, min((uint32_t)b, m));
}

// Any strides and alignments: 64 x 64 tiles of C, 64 bytes of k at a time in
// shared memory, 4 x 4 cells a thread with the 4-way byte product.
constexpr int TM = 64, TN = 64, TK = 64, kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) mm_i8_tile_kernel(const MapalI8Site S, const int8_t* __restrict__ A,
                                                              const float* __restrict__ sa,
                                                              const int8_t* __restrict__ B,
                                                              const float* __restrict__ sb,
                                                              const int32_t* __restrict__ offsets, T* __restrict__ C,
                                                              unsigned* trap) {
  __shared__ __align__(16) int8_t ta[TM][TK + 4], tb[TN][TK + 4];
  uint32_t lo = 0, hi = (uint32_t)S.m;
  const uint32_t g = blockIdx.z;
  if (offsets) group_rows(offsets, g, (uint32_t)S.m, trap, lo, hi);
  const uint64_t n0 = (uint64_t)blockIdx.x * TN;
  const int8_t* Bg = B + g * S.ldg;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (uint64_t m0 = lo + (uint64_t)blockIdx.y * TM; m0 < hi; m0 += (uint64_t)gridDim.y * TM) {
    int acc[4][4] = {};
    for (uint64_t k0 = 0; k0 < S.k; k0 += TK) {
      __syncthreads();
      for (int i = threadIdx.x; i < TM * TK; i += kThreads) {
        const int r = i / TK, c = i % TK;
        const bool in = k0 + c < S.k;
        ta[r][c] = in && m0 + r < hi ? A[(m0 + r) * S.lda + k0 + c] : (int8_t)0;
        tb[r][c] = in && n0 + r < S.n ? Bg[(n0 + r) * S.ldb + k0 + c] : (int8_t)0;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < TK; kk += 4) {
        int a[4], b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          a[u] = *reinterpret_cast<const int*>(&ta[ty + 16 * u][kk]);
          b[u] = *reinterpret_cast<const int*>(&tb[tx + 16 * u][kk]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[u][v] = __dp4a(a[u], b[v], acc[u][v]);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const uint64_t i = m0 + ty + 16 * u, j = n0 + tx + 16 * v;
        if (i < hi && j < S.n)
          C[i * S.ldc + j] = scaled<T>(acc[u][v], sa ? sa[i] : 1.0f, sb ? sb[g * S.n + j] : 1.0f);
      }
  }
}

int check_site(const MapalI8Site* s) {
  if (!s) return set_error(MAPAL_ERR_INVALID, "site is null");
  const int es = dtype_bytes(s->dtype);
  if (es < 2) return set_error(MAPAL_ERR_INVALID, "C is f32, f16 or bf16");
  if (s->groups == 0 || s->groups > 65535) return set_error(MAPAL_ERR_INVALID, "1 to 65535 groups");
  if (s->k >= 131072) return set_error(MAPAL_ERR_UNSUPPORTED, "k of 131072 or more: a sum could leave 32 bits");
  if (s->m > 0x7fffffffull || s->n > 0x7fffffffull) return set_error(MAPAL_ERR_UNSUPPORTED, "m or n of 2^31 or more");
  if (!rows_ok(s->m, s->k, s->lda, 1) || !rows_ok(s->n, s->k, s->ldb, 1) || !rows_ok(s->m, s->n, s->ldc, es))
    return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
  const uint64_t one = s->n ? (s->n - 1) * s->ldb + s->k : 0;
  if (s->groups > 1 && !rows_ok(s->groups, one, s->ldg, 1))
    return set_error(MAPAL_ERR_INVALID, "the stride between groups is shorter than a matrix, or too long");
  return 0;
}

template <typename T>
int launch_tiles(const DeviceSlot& D, const MapalI8Site& s, const int8_t* A, const float* sa, const int8_t* B,
                 const float* sb, const int32_t* offsets, void* C) {
  const uint64_t bx = (s.n + TN - 1) / TN, rows = (s.m + TM - 1) / TM;
  const uint64_t cap = s.groups > 1 ? 64 : 65535;  // row tiles beyond the grid are walked by its blocks
  mm_i8_tile_kernel<T><<<dim3((unsigned)bx, (unsigned)(rows < cap ? rows : cap), s.groups), kThreads, 0, D.stream>>>(
      s, A, sa, B, sb, offsets, (T*)C, D.trap);
  count_launch();
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
    MAPAL_TRY(enter(ctx));
    DeviceSlot& D = ctx->dev[0];
    int rc;
    if (s.dtype == MAPAL_DTYPE_F32)
      rc = launch_tiles<float>(D, s, A, scale_a, B, scale_b, offsets, C);
    else if (s.dtype == MAPAL_DTYPE_F16)
      rc = launch_tiles<__half>(D, s, A, scale_a, B, scale_b, offsets, C);
    else
      rc = launch_tiles<__nv_bfloat16>(D, s, A, scale_a, B, scale_b, offsets, C);
    MAPAL_TRY(rc);
    return finish(ctx, 0, offsets != nullptr);
  });
}

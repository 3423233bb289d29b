// quant.cu — rows to 8 bits with a scale each (mapal_gpu_quantize_rows_i8).
// No counterpart in the reference.
//
// a = max|x|, scale = a/127, q = clamp(rint(x*(127/a)), -127, 127). The
// maximum is taken over the bit patterns of |x| as integers, which order as
// the values do with infinity and then NaN above them, so one reduction finds
// the maximum and whether the row is finite.
#include "rows.cuh"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInf = 0x7f800000u;

struct RowScale {
  float inv;    // 127/a, or 0 for a row that becomes zeros
  float scale;  // a/127
};

__device__ __forceinline__ RowScale row_scale(uint32_t most) {
  RowScale r;
  const float a = __uint_as_float(most);
  r.inv = __fdiv_rn(127.0f, a);
  r.scale = __fdiv_rn(a, 127.0f);
  if (most >= kInf) {
    r.inv = 0.0f;
    r.scale = __uint_as_float(0x7fffffffu);
  } else if (!(r.inv < __uint_as_float(kInf))) {
    r.inv = 0.0f;
    r.scale = 0.0f;
  }
  return r;
}

// A finite row's value; a row with inv = 0 gives 0 whatever x is.
__device__ __forceinline__ int8_t quantized(float x, float inv) {
  const float v = inv == 0.0f ? 0.0f : rintf(__fmul_rn(x, inv));
  return (int8_t)fminf(fmaxf(v, -127.0f), 127.0f);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
}

// One block a row, two passes over it.
template <typename T>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(const MapalQuantSite S, const T* x, int8_t* q,
                                                              float* scale) {
  __shared__ uint32_t red[2][32];
  int par = 0;
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x, par ^= 1) {
    const T* xr = x + r * S.ldx;
    uint32_t most = 0;
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads) most = max(most, __float_as_uint(to_f32(xr[i])) & 0x7fffffffu);
    const RowScale rs = row_scale(block_max(most, red[par]));
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads) q[r * S.ldq + i] = quantized(to_f32(xr[i]), rs.inv);
    if (threadIdx.x == 0) scale[r] = rs.scale;
  }
}

template <typename T>
void launch_quant(const DeviceSlot& D, const MapalQuantSite& s, const void* x, int8_t* q, float* scale) {
  const unsigned grid = (unsigned)(s.rows < 8ull * D.prof.sm_count ? s.rows : 8ull * D.prof.sm_count);
  quant_rows_kernel<T><<<grid, kThreads, 0, D.stream>>>(s, (const T*)x, q, scale);
  count_launch();
}

}  // namespace

extern "C" int mapal_gpu_quantize_rows_i8(MapalGpuCtx* ctx, const MapalQuantSite* site, const void* x, int8_t* q,
                                          float* scale) {
  return guarded([&]() -> int {
    if (!site) return set_error(MAPAL_ERR_INVALID, "site is null");
    const int es = dtype_bytes(site->dtype);
    if (es < 2) return set_error(MAPAL_ERR_INVALID, "rows of f32, f16 or bf16 are quantised");
    if (site->d > 0x7fffffffull || !rows_ok(site->rows, site->d, site->ldx, es) ||
        !rows_ok(site->rows, site->d, site->ldq, 1))
      return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
    if (site->rows == 0) return 0;
    if (!scale || (site->d && (!x || !q))) return set_error(MAPAL_ERR_INVALID, "null x, q or scale");
    if (((uintptr_t)x & (es - 1)) || ((uintptr_t)scale & 3))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    MAPAL_TRY(enter(ctx));
    if (site->dtype == MAPAL_DTYPE_F32)
      launch_quant<float>(ctx->dev[0], *site, x, q, scale);
    else if (site->dtype == MAPAL_DTYPE_F16)
      launch_quant<__half>(ctx->dev[0], *site, x, q, scale);
    else
      launch_quant<__nv_bfloat16>(ctx->dev[0], *site, x, q, scale);
    return finish(ctx, 0, false);
  });
}

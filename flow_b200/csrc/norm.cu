// norm.cu — layer norm over rows, forward and backward (mapal_gpu_layer_norm,
// mapal_gpu_layer_norm_grad). No counterpart in the reference.
//
// Forward: mu = mean(x), r = 1/sqrt(mean((x - mu)^2) + eps), y = (x - mu)*r*w + b.
// Backward, with h = (x - mu)*r and g = dy*w:
//   dx = r*(g - mean(g) - h*mean(g*h)), dw = sum_rows dy*h, db = sum_rows dy.
#include "rows.cuh"

namespace {

constexpr int kThreads = 256;

template <typename TW>
__device__ __forceinline__ float weight_at(const void* w, uint64_t i, float none) {
  return w ? to_f32(static_cast<const TW*>(w)[i]) : none;
}

__device__ __forceinline__ float inv_std(float var, float eps) { return __fdiv_rn(1.0f, __fsqrt_rn(var + eps)); }

// One block a row, three passes over it.
template <typename T, typename TW>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(const MapalNormSite S, const T* x, const void* w,
                                                             const void* b, T* y, float* mean, float* rstd) {
  __shared__ float red[2][32];
  const float n = (float)S.d;
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x) {
    const T* xr = x + r * S.ldx;
    T* yr = y + r * S.ldy;
    float s = 0.0f;
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads) s += to_f32(xr[i]);
    const float mu = __fdiv_rn(block_sum(s, red[0]), n);
    float q = 0.0f;
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads) {
      const float c = to_f32(xr[i]) - mu;
      q = __fmaf_rn(c, c, q);
    }
    const float rs = inv_std(__fdiv_rn(block_sum(q, red[1]), n), S.eps);
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads)
      yr[i] = from_f32<T>(
          __fmaf_rn((to_f32(xr[i]) - mu) * rs, weight_at<TW>(w, i, 1.0f), weight_at<TW>(b, i, 0.0f)));
    if (threadIdx.x == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

// One block a row: the row's two means, then dx.
template <typename T, typename TW>
__global__ void __launch_bounds__(kThreads) norm_grad_rows_kernel(const MapalNormSite S, const T* x, const void* w,
                                                                  const float* mean, const float* rstd, const T* dy,
                                                                  T* dx) {
  __shared__ float red[2][2][32];
  const float n = (float)S.d;
  int par = 0;
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x, par ^= 1) {
    const T* xr = x + r * S.ldx;
    const T* dyr = dy + r * S.lddy;
    T* dxr = dx + r * S.lddx;
    const float mu = mean[r], rs = rstd[r];
    float c1 = 0.0f, c2 = 0.0f;
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads) {
      const float g = to_f32(dyr[i]) * weight_at<TW>(w, i, 1.0f);
      c1 += g;
      c2 = __fmaf_rn(g, (to_f32(xr[i]) - mu) * rs, c2);
    }
    c1 = __fdiv_rn(block_sum(c1, red[par][0]), n);
    c2 = __fdiv_rn(block_sum(c2, red[par][1]), n);
    for (uint64_t i = threadIdx.x; i < S.d; i += kThreads) {
      const float g = to_f32(dyr[i]) * weight_at<TW>(w, i, 1.0f);
      const float h = (to_f32(xr[i]) - mu) * rs;
      dxr[i] = from_f32<T>((g - c1 - h * c2) * rs);
    }
  }
}

// dw and db over rows p, p + parts, ...: part p writes its sums of 32 columns.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_grad_cols_kernel(const MapalNormSite S, const T* x, const float* mean,
                                                                  const float* rstd, const T* dy, float* work,
                                                                  uint32_t parts) {
  __shared__ float sw[8][32], sb[8][32];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float aw = 0.0f, ab = 0.0f;
  if (c < S.d)
    for (uint64_t r = blockIdx.y * 8ull + sub; r < S.rows; r += parts * 8ull) {
      const float g = to_f32(dy[r * S.lddy + c]);
      aw = __fmaf_rn(g, (to_f32(x[r * S.ldx + c]) - mean[r]) * rstd[r], aw);
      ab += g;
    }
  sw[sub][lane] = aw;
  sb[sub][lane] = ab;
  __syncthreads();
  if (sub == 0 && c < S.d) {
    for (int k = 1; k < 8; ++k) {
      aw += sw[k][lane];
      ab += sb[k][lane];
    }
    work[(2ull * blockIdx.y) * S.d + c] = aw;
    work[(2ull * blockIdx.y + 1) * S.d + c] = ab;
  }
}

// dw and db from the parts' sums, in part order.
__global__ void __launch_bounds__(kThreads) norm_grad_join_kernel(const float* work, uint64_t d, uint32_t parts,
                                                                  float* dw, float* db) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;  // 0..d: dw, d..2d: db
  float a = 0.0f;
  if (c < 2 * d)
    for (uint32_t p = sub; p < parts; p += 8) a += work[2ull * p * d + c];
  red[sub][lane] = a;
  __syncthreads();
  if (sub == 0 && c < 2 * d) {
    for (int k = 1; k < 8; ++k) a += red[k][lane];
    float* out = c < d ? dw : db;
    if (out) out[c < d ? c : c - d] = a;
  }
}

int check_norm(const MapalNormSite* s) {
  if (!s) return set_error(MAPAL_ERR_INVALID, "site is null");
  const int es = dtype_bytes(s->dtype);
  if (es == 0 || s->dtype == MAPAL_DTYPE_I8) return set_error(MAPAL_ERR_INVALID, "layer norm takes f32, f16 or bf16");
  if (s->wtype != s->dtype && s->wtype != MAPAL_DTYPE_F32)
    return set_error(MAPAL_ERR_INVALID, "the weight's type is the rows' or f32");
  if (s->d == 0 || s->d > 0x7fffffffull) return set_error(MAPAL_ERR_INVALID, "rows of 1 to 2^31 - 1 elements");
  if (!(s->eps >= 0.0f)) return set_error(MAPAL_ERR_INVALID, "eps is negative or NaN");
  return 0;
}

uint32_t grad_parts(const MapalNormSite& s, int sms) {
  const uint64_t want = (s.rows + 7) / 8, cap = 2ull * sms;
  return (uint32_t)(want < 1 ? 1 : want < cap ? want : cap);
}

uint64_t grad_bytes(const MapalNormSite& s, int sms) { return grad_parts(s, sms) * 2ull * s.d * sizeof(float); }

template <typename T, typename TW>
void launch_norm(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const void* b, void* y,
                 float* mean, float* rstd) {
  const unsigned grid = (unsigned)(s.rows < 8ull * D.prof.sm_count ? s.rows : 8ull * D.prof.sm_count);
  norm_rows_kernel<T, TW><<<grid, kThreads, 0, D.stream>>>(s, (const T*)x, w, b, (T*)y, mean, rstd);
  count_launch();
}

template <typename T, typename TW>
int launch_norm_grad(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const float* mean,
                     const float* rstd, const void* dy, void* dx, float* dw, float* db, float* work) {
  const uint32_t parts = grad_parts(s, D.prof.sm_count);
  const unsigned blocks = (unsigned)((s.d + 31) / 32);
  if (dw || db) {
    norm_grad_cols_kernel<T><<<dim3(blocks, parts), kThreads, 0, D.stream>>>(s, (const T*)x, mean, rstd,
                                                                             (const T*)dy, work, parts);
    count_launch();
    norm_grad_join_kernel<<<(unsigned)((2 * s.d + 31) / 32), kThreads, 0, D.stream>>>(work, s.d, parts, dw, db);
    count_launch();
  }
  if (s.rows) {
    const unsigned grid = (unsigned)(s.rows < 8ull * D.prof.sm_count ? s.rows : 8ull * D.prof.sm_count);
    norm_grad_rows_kernel<T, TW><<<grid, kThreads, 0, D.stream>>>(s, (const T*)x, w, mean, rstd, (const T*)dy, (T*)dx);
    count_launch();
  }
  return 0;
}

// f(T, TW) for the site's types.
template <typename F>
auto by_type(const MapalNormSite& s, F&& f) {
  const bool wide = s.wtype == MAPAL_DTYPE_F32;
  if (s.dtype == MAPAL_DTYPE_F32) return f(float{}, float{});
  if (s.dtype == MAPAL_DTYPE_F16) return wide ? f(__half{}, float{}) : f(__half{}, __half{});
  return wide ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace

extern "C" int mapal_gpu_layer_norm(MapalGpuCtx* ctx, const MapalNormSite* site, const void* x, const void* w,
                                    const void* b, void* y, float* mean, float* rstd) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_norm(site));
    const int es = dtype_bytes(site->dtype), ws = dtype_bytes(site->wtype);
    if (!rows_ok(site->rows, site->d, site->ldx, es) || !rows_ok(site->rows, site->d, site->ldy, es))
      return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
    if (site->rows == 0) return 0;
    if (!x || !y) return set_error(MAPAL_ERR_INVALID, "null x or y");
    if (!aligned_to(x, es) || !aligned_to(y, es) || !aligned_to(w, ws) || !aligned_to(b, ws) ||
        !aligned_to(mean, 4) || !aligned_to(rstd, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    MAPAL_TRY(enter(ctx));
    by_type(*site, [&](auto t, auto tw) {
      launch_norm<decltype(t), decltype(tw)>(ctx->dev[0], *site, x, w, b, y, mean, rstd);
      return 0;
    });
    return finish(ctx, 0, false);
  });
}

extern "C" int mapal_gpu_layer_norm_grad_workspace(MapalGpuCtx* ctx, const MapalNormSite* site, uint64_t* bytes) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_norm(site));
    if (!bytes) return set_error(MAPAL_ERR_INVALID, "bytes is null");
    MAPAL_TRY(enter(ctx));
    *bytes = grad_bytes(*site, ctx->dev[0].prof.sm_count);
    return 0;
  });
}

extern "C" int mapal_gpu_layer_norm_grad(MapalGpuCtx* ctx, const MapalNormSite* site, const void* x, const void* w,
                                         const float* mean, const float* rstd, const void* dy, void* dx, float* dw,
                                         float* db, void* work, uint64_t work_bytes) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_norm(site));
    const int es = dtype_bytes(site->dtype), ws = dtype_bytes(site->wtype);
    if (!rows_ok(site->rows, site->d, site->ldx, es) || !rows_ok(site->rows, site->d, site->lddy, es) ||
        !rows_ok(site->rows, site->d, site->lddx, es))
      return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
    if (site->rows && (!x || !mean || !rstd || !dy || !dx))
      return set_error(MAPAL_ERR_INVALID, "null x, mean, rstd, dy or dx");
    if (!aligned_to(x, es) || !aligned_to(dy, es) || !aligned_to(dx, es) || !aligned_to(w, ws) ||
        !aligned_to(mean, 4) || !aligned_to(rstd, 4) || !aligned_to(dw, 4) || !aligned_to(db, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    if ((dw || db) && (!work || !aligned16(work)))
      return set_error(MAPAL_ERR_INVALID, "work is null or not 16-byte aligned");
    if (site->rows == 0 && !dw && !db) return 0;
    MAPAL_TRY(enter(ctx));
    if ((dw || db) && work_bytes < grad_bytes(*site, ctx->dev[0].prof.sm_count))
      return set_error(MAPAL_ERR_INVALID, "work is shorter than mapal_gpu_layer_norm_grad_workspace says");
    MAPAL_TRY(by_type(*site, [&](auto t, auto tw) {
      return launch_norm_grad<decltype(t), decltype(tw)>(ctx->dev[0], *site, x, w, mean, rstd, dy, dx, dw, db,
                                                         (float*)work);
    }));
    return finish(ctx, 0, false);
  });
}

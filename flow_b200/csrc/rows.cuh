// rows.cuh — what the row-wise operators (layer norm, expert rows, 8-bit rows
// and products) share: element types, vector loads, row reductions and the
// checks of their records. Not part of the ABI.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <exception>

#include "common.cuh"

// ---- element types ----------------------------------------------------------------

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// One rounding to nearest even, at the end of an operator's f32 arithmetic.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V elements moved as one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

inline int dtype_bytes(int dtype) {
  return dtype == MAPAL_DTYPE_F32 ? 4 : dtype == MAPAL_DTYPE_F16 || dtype == MAPAL_DTYPE_BF16 ? 2 : dtype == MAPAL_DTYPE_I8 ? 1 : 0;
}

// ---- reductions -------------------------------------------------------------------

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The sum over a block of whole warps, in every thread. `red` holds 32 floats;
// a caller that reduces twice without a barrier in between passes another 32.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? red[lane] : 0.0f);
}

// ---- entry points -----------------------------------------------------------------

// The caller's current device is put back when an entry point returns.
struct DeviceGuard {
  int prev = -1;
  DeviceGuard() {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// No C++ exception leaves an entry point (the error text is a std::string).
template <typename F>
int guarded(F&& f) noexcept {
  try {
    DeviceGuard g;
    return f();
  } catch (...) {
    return MAPAL_ERR_NOMEM;
  }
}

// rows x cols elements at row stride ld: the stride covers a row, and the last
// byte's offset fits in 62 bits.
inline bool rows_ok(uint64_t rows, uint64_t cols, uint64_t ld, uint64_t elem) {
  if (rows > 1 && ld < cols) return false;
  const uint64_t lim = 1ull << 62;
  if (cols > lim / elem) return false;
  if (rows <= 1 || ld == 0) return true;
  return ld <= lim / elem && (rows - 1) <= (lim / elem - cols) / ld;
}

// The widest access of 16, 8, 4, 2 or 1 bytes that a pointer and a row stride
// (in bytes; ignored for a single row) are multiples of.
inline int align_of(const void* p, uint64_t stride_bytes, uint64_t rows) {
  const uint64_t v = (uint64_t)(uintptr_t)p | (rows > 1 ? stride_bytes : 0) | 16u;
  return (int)(v & (~v + 1));
}

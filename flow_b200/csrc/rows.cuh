// rows.cuh — what the row-wise operators (layer norm, expert rows, 8-bit rows
// and products) share: element types, vector loads, row reductions and the
// checks of their records. Not part of the ABI.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string.h>

#include <exception>
#include <type_traits>

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

// V elements moved as one access, held as 32-bit words (or one 16-bit value).
// Converted a word at a time: two bf16 are a shift and a mask, and pairs are
// rounded by one instruction.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  static constexpr int W = sizeof(T) * V / 4;  // 0: a single 16-bit element
  using Word = std::conditional_t<W == 0, uint16_t, uint32_t>;
  Word w[W == 0 ? 1 : W];

  __device__ __forceinline__ void get(float (&f)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      if constexpr (W == 0) {
        f[0] = __uint_as_float((uint32_t)w[0] << 16);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    } else {
      if constexpr (W == 0) {
        f[0] = __half2float(__ushort_as_half(w[0]));
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          __half2 h;
          memcpy(&h, &w[i], 4);
          const float2 g = __half22float2(h);
          f[2 * i] = g.x;
          f[2 * i + 1] = g.y;
        }
      }
    }
  }

  __device__ __forceinline__ void set(const float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else if constexpr (W == 0) {
      const T v = from_f32<T>(f[0]);
      memcpy(&w[0], &v, 2);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          memcpy(&w[i], &v, 4);
        } else {
          const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          memcpy(&w[i], &v, 4);
        }
      }
    }
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (W == 0 ? 1 : W); ++i) w[i] = 0;
  }

  // Zeros for the elements whose bits are not in m.
  __device__ __forceinline__ void keep(uint32_t m) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = m & (1u << i) ? w[i] : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i)
        w[i] &= (m & (1u << (2 * i)) ? 0xffffu : 0u) | (m & (2u << (2 * i)) ? 0xffff0000u : 0u);
    }
  }

  // Hides where the bits come from, so that a later use converts them again
  // instead of keeping the floats of an earlier one in registers.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < (W == 0 ? 1 : W); ++i) {
      if constexpr (W == 0)
        asm volatile("" : "+h"(w[i]));
      else
        asm volatile("" : "+r"(w[i]));
    }
  }
};

// A pack read or written once (no reuse expected in this kernel).
template <typename P>
__device__ __forceinline__ P ld_once(const P* p) {
  P r;
  if constexpr (sizeof(P) == 16) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (sizeof(P) == 4) {
    r.w[0] = __ldcs(reinterpret_cast<const unsigned*>(p));
  } else {
    static_assert(sizeof(P) == 2, "packs of 2, 4 or 16 bytes");
    r.w[0] = __ldcs(reinterpret_cast<const unsigned short*>(p));
  }
  return r;
}
template <typename P>
__device__ __forceinline__ void st_once(P* p, const P& r) {
  if constexpr (sizeof(P) == 16) {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]));
  } else if constexpr (sizeof(P) == 4) {
    __stcs(reinterpret_cast<unsigned*>(p), r.w[0]);
  } else {
    static_assert(sizeof(P) == 2, "packs of 2, 4 or 16 bytes");
    __stcs(reinterpret_cast<unsigned short*>(p), r.w[0]);
  }
}

// The elements of a pack whose bits are in m, one by one.
template <typename T, int V>
__device__ __forceinline__ void st_part(T* p, const Pack<T, V>& r, uint32_t m) {
  T v[V];
  memcpy(v, r.w, sizeof(v));
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (m & (1u << e)) p[e] = v[e];
}

// Bytes sh..sh+15 of a (first) and b.
__device__ __forceinline__ uint4 straddle(const uint4& a, const uint4& b, uint32_t sh) {
  const bool by8 = sh & 8, by4 = sh & 4;
  const uint32_t bits = (sh & 3) * 8;
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = by8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = by4 ? w[i + 1] : w[i];
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

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

// ---- launches ---------------------------------------------------------------------
//
// The kernels of the row-wise operators may be launched before the kernel ahead
// of them in the stream has finished (programmatic stream serialization): each
// does what needs no memory of others, then waits for it with grid_wait, before
// its first access to global memory, and lets the next one in with grid_go. In a
// row of short kernels that hides a launch and a prologue, 1 to 1.5 us each.

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
int launch_rows(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, unsigned cluster,
                A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  MAPAL_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
  count_launch();
  return 0;
}

// ---- entry points -----------------------------------------------------------------

// The context's first device is current while this lives; the caller's current
// device is put back after. Nothing is set where the two are the same, which
// spares a small call two of its driver calls.
struct OnDevice {
  int prev = -1, rc;
  explicit OnDevice(MapalGpuCtx* ctx) {
    int cur = -1;
    if (ctx && cudaGetDevice(&cur) == cudaSuccess && cur == ctx->dev[0].device) {
      rc = 0;
      return;
    }
    prev = cur;
    rc = enter(ctx);
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
};

// No C++ exception leaves an entry point (the error text is a std::string).
template <typename F>
int guarded(F&& f) noexcept {
  try {
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

// `bytes` of each of some rows copied, or set to zeros (from null), at strides in bytes.
// One row's stride may be anything, and the runtime's own two-dimensional calls take
// strides up to 2^31 - 1: longer ones are some hundred rows at most in a device's memory.
inline int copy_rows(void* to, uint64_t ldt, const void* from, uint64_t ldf, uint64_t bytes, uint64_t rows, cudaStream_t stream) {
  if (rows <= 1 || (ldt == bytes && (!from || ldf == bytes))) {
    bytes *= rows;
    rows = 1;
    ldt = ldf = bytes;
  }
  const uint64_t most = 0x7fffffff;
  if (rows > 1 && ldt <= most && (!from || ldf <= most)) {
    if (from)
      MAPAL_CUDA(cudaMemcpy2DAsync(to, ldt, from, ldf, bytes, rows, cudaMemcpyDeviceToDevice, stream));
    else
      MAPAL_CUDA(cudaMemset2DAsync(to, ldt, 0, bytes, rows, stream));
    return 0;
  }
  for (uint64_t r = 0; r < rows; ++r) {
    uint8_t* p = static_cast<uint8_t*>(to) + r * ldt;
    if (from)
      MAPAL_CUDA(cudaMemcpyAsync(p, static_cast<const uint8_t*>(from) + r * ldf, bytes, cudaMemcpyDeviceToDevice, stream));
    else
      MAPAL_CUDA(cudaMemsetAsync(p, 0, bytes, stream));
  }
  return 0;
}

// The widest access of 16, 8, 4, 2 or 1 bytes that a pointer and a row stride
// (in bytes; ignored for a single row) are multiples of.
inline int align_of(const void* p, uint64_t stride_bytes, uint64_t rows) {
  const uint64_t v = (uint64_t)(uintptr_t)p | (rows > 1 ? stride_bytes : 0) | 16u;
  return (int)(v & (~v + 1));
}

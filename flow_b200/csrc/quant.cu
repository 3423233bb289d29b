// quant.cu — rows to 8 bits with a scale each (mapal_gpu_quantize_rows_i8).
// No counterpart in the reference.
//
// a = max|x|, scale = a/127, q = clamp(rint(x*(127/a)), -127, 127). The
// maximum is taken over the bit patterns of |x| as integers, which order as
// the values do with infinity and then NaN above them, so one reduction finds
// the maximum and whether the row is finite.
//
// Bound by HBM (an element's bytes and one), so a row is read once and held in
// registers as it came, and the instructions an element are kept few: the
// maximum of 16-bit types is taken on pairs, one redux instruction joins a
// warp, and rint is an addition of 1.5*2^23, after which the low byte is the
// integer.
#include "f32x2.cuh"
#include "rowflow.cuh"

namespace {

constexpr uint32_t kInf = 0x7f800000u;

struct RowScale {
  float inv;    // 127/a, or 0 for a row that becomes zeros
  float scale;  // a/127
};

// From the largest |x| as the bits of a float.
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

// The largest |x| of what a thread has seen, as the bits of a value of T: one
// word, or two 16-bit halves.
template <typename T>
struct Most {
  uint32_t m = 0;
  template <int V>
  __device__ __forceinline__ void add(const Pack<T, V>& p) {
    using P = Pack<T, V>;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < P::W; ++i) m = max(m, p.w[i] & 0x7fffffffu);
    } else if constexpr (P::W == 0) {
      m = max(m, (uint32_t)p.w[0] & 0x7fffu);
    } else {
#pragma unroll
      for (int i = 0; i < P::W; ++i) m = __vmaxu2(m, p.w[i] & 0x7fff7fffu);
    }
  }
  // As one value of T's bits.
  __device__ __forceinline__ uint32_t bits() const { return sizeof(T) == 4 ? m : max(m >> 16, m & 0xffffu); }
};

template <typename T>
__device__ __forceinline__ uint32_t float_bits(uint32_t b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return b << 16;
  if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)b)));
  return b;
}

// V values of a finite row: |x*inv| is at most 127 (and a rounding), so the
// sum with 1.5*2^23 holds the integer in its low byte, rounded to nearest even
// by the addition. The product is rounded before (packed products would be
// fused with the addition).
template <typename T, int V>
__device__ __forceinline__ void quantize(const Pack<T, V>& p, float inv, uint32_t (&out)[V >= 4 ? V / 4 : 1]) {
  const f2 magic = f2_splat(12582912.0f);
  float f[V];
  p.get(f);
  uint32_t b[V];
  if constexpr (V > 1) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const f2 v = f2_add(f2_pack(__fmul_rn(f[e], inv), __fmul_rn(f[e + 1], inv)), magic);
      b[e] = __float_as_uint(f2_lo(v));
      b[e + 1] = __float_as_uint(f2_hi(v));
    }
  } else {
    b[0] = __float_as_uint(__fadd_rn(__fmul_rn(f[0], inv), 12582912.0f));
  }
  // a row of zeros: whatever x was (a NaN times 0 is a NaN)
  const uint32_t keep = inv == 0.0f ? 0u : 0xffffffffu;
  if constexpr (V >= 4) {
#pragma unroll
    for (int e = 0; e < V; e += 4)
      out[e / 4] = __byte_perm(__byte_perm(b[e], b[e + 1], 0x0040), __byte_perm(b[e + 2], b[e + 3], 0x0040), 0x5410) & keep;
  } else if constexpr (V == 2) {
    out[0] = __byte_perm(b[0], b[1], 0x0040) & keep;
  } else {
    out[0] = b[0] & keep;
  }
}

template <int V>
__device__ __forceinline__ void put(int8_t* q, const uint32_t (&o)[V >= 4 ? V / 4 : 1]) {
  if constexpr (V == 8)
    __stcs(reinterpret_cast<uint2*>(q), make_uint2(o[0], o[1]));
  else if constexpr (V == 4)
    __stcs(reinterpret_cast<unsigned*>(q), o[0]);
  else if constexpr (V == 2)
    __stcs(reinterpret_cast<unsigned short*>(q), (unsigned short)o[0]);
  else
    __stcs(reinterpret_cast<unsigned char*>(q), (unsigned char)o[0]);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
}

// ROWS rows at a time through the ring, a group of warps with EACH elements a
// thread: rows that fit in a block's registers.
template <typename T, int V, int EACH, int ROWS, int EDGE>
__global__ void __launch_bounds__(kFlow, 1) quant_flow_kernel(const MapalQuantSite S, const T* x, int8_t* q, float* scale,
                                                              int group, uint32_t period) {
  using R = std::conditional_t<EDGE != 0, EdgeRing<T, EACH, ROWS, 1, false, EDGE == 2>, Ring<T, V, EACH, ROWS, 1>>;
  using P = Pack<T, V>;
  constexpr int NV = EACH / V;
  __shared__ uint32_t sets[kFlow / 32][2][ROWS][16];
  extern __shared__ __align__(16) uint8_t dyn[];
  const Group<false> G(group);
  R ring(dyn, G);
  const int d = (int)S.d, lane = threadIdx.x & 31, warps = group / 32;
  const Turns<false, EDGE, ROWS> mine(G, period, S.rows);
  uint64_t rows = mine.rows, ldx = mine.stride(S.ldx), ldq = mine.stride(S.ldq), r = mine.first;
  const int shift = mine.template shift<T>(S.ldq), shift_x = mine.template shift<T>(S.ldx);
  const std::conditional_t<EDGE != 0, Input<V, NV>, Whole> in(group, G.tid, d, shift_x, shift);
  const std::conditional_t<EDGE != 0, Mine<V, NV>, Whole> part(group, G.tid, shift, d + shift);
  const std::conditional_t<EDGE != 0, Masks<P, V, NV>, Whole> keep(part);
  x = mine.at(x, S.ldx) - shift_x + (G.tid - in.back) * V;
  q = mine.at(q, S.ldq) - shift + G.tid * V;
  scale = mine.at(scale, 1);
  if constexpr (EDGE != 0) {
    pin(x), pin(q), pin(scale);
    pin(rows), pin(ldx), pin(ldq);
  }
  auto start = [&](int st, uint64_t row) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (row + k < rows) {
        const T* from = x + (row + k) * ldx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if constexpr (EDGE != 0)
            ring.bring(st, k * NV + j, from + j * group * V, in.left[j]);
          else if ((j * group + G.tid) * V < d)
            ring.copy(st, k * NV + j, from + j * group * V);
        }
      }
    ring.commit();
  };
  grid_wait();
  grid_go();
#pragma unroll
  for (int k = 0; k < R::kStages; ++k) start(k, r + k * mine.step);
  for (int par = 0; r < rows; r += mine.step, par ^= 1) {
    ring.wait();
    P v[ROWS][NV];
    uint32_t most[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      Most<T> m;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (EDGE != 0) {
          v[k][j] = ring.take(k * NV + j, in.by);
          keep(v[k][j], j);
        } else if ((j * group + G.tid) * V < d && r + k < rows) {
          v[k][j] = ring.take(k * NV + j);
        } else {
          v[k][j].clear();
        }
        m.add(v[k][j]);
      }
      most[k] = __reduce_max_sync(0xffffffffu, m.bits());
    }
    if constexpr (EDGE != 0) ring.taken();
    start(ring.stage, r + R::kStages * mine.step);  // this turn's slots have been read
    ring.next_stage();
    if (warps > 1) {
      auto* red = sets[G.id][par];
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < ROWS; ++k) red[k][G.tid >> 5] = most[k];
      G.sync();
#pragma unroll
      for (int k = 0; k < ROWS; ++k) most[k] = __reduce_max_sync(0xffffffffu, lane < warps ? red[k][lane] : 0u);
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (r + k >= rows) break;
      const RowScale rs = row_scale(float_bits<T>(most[k]));
      int8_t* to = q + (r + k) * ldq;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint32_t o[V >= 4 ? V / 4 : 1];
        quantize<T, V>(v[k][j], rs.inv, o);
        if constexpr (EDGE != 0) {
          if (part.at(j) == part.kAll) {
            put<V>(to + j * group * V, o);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (part.at(j) & (1u << e)) to[j * group * V + e] = (int8_t)(o[e / 4] >> (8 * (e % 4)));
          }
        } else if ((j * group + G.tid) * V < d) {
          put<V>(to + j * group * V, o);
        }
      }
      if (G.tid == 0) scale[(r + k) * mine.period] = rs.scale;
    }
  }
}

// One block a row. EACH elements a thread are held from the first pass to the
// second; EACH 0: any length, read twice.
template <typename T, int V, int EACH>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const MapalQuantSite S, const T* x, int8_t* q, float* scale) {
  using P = Pack<T, V>;
  constexpr int NV = EACH ? EACH / V : 1;
  __shared__ uint32_t red[2][32];
  const int64_t d = (int64_t)S.d, step = (int64_t)blockDim.x * V;
  int par = 0;
  grid_wait();
  grid_go();
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x, par ^= 1) {
    const T* xr = x + r * S.ldx;
    P v[NV];
    Most<T> m;
    if constexpr (EACH > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int64_t i = threadIdx.x * V + j * step;
        if (i < d)
          v[j] = ld_once(reinterpret_cast<const P*>(xr + i));
        else
          v[j].clear();
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) m.add(v[j]);
    } else {
#pragma unroll 4
      for (int64_t i = threadIdx.x * V; i < d; i += step) m.add(*reinterpret_cast<const P*>(xr + i));
    }
    const RowScale rs = row_scale(float_bits<T>(block_max(m.bits(), red[par])));
    uint32_t o[V >= 4 ? V / 4 : 1];
    if constexpr (EACH > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int64_t i = threadIdx.x * V + j * step;
        quantize<T, V>(v[j], rs.inv, o);
        if (i < d) put<V>(q + r * S.ldq + i, o);
      }
    } else {
#pragma unroll 4
      for (int64_t i = threadIdx.x * V; i < d; i += step) {
        quantize<T, V>(*reinterpret_cast<const P*>(xr + i), rs.inv, o);
        put<V>(q + r * S.ldq + i, o);
      }
    }
    if (threadIdx.x == 0) scale[r] = rs.scale;
  }
}

template <typename T, int V, int EACH, int ROWS, int EDGE = 0>
int launch_flow(const DeviceSlot& D, const MapalQuantSite& s, const T* x, int8_t* q, float* scale) {
  constexpr size_t smem =
      std::conditional_t<EDGE != 0, EdgeRing<T, EACH, ROWS, 1, false, EDGE == 2>, Ring<T, V, EACH, ROWS, 1>>::kBytes;
  static std::atomic<uint64_t> done{0};
  auto kernel = quant_flow_kernel<T, V, EACH, ROWS, EDGE>;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, smem, "quantize_rows shared memory"));
  const uint32_t period = EDGE ? edge_period(s.rows, {s.ldx, s.ldq}, V) : 1;
  const Plan p = flow_plan<false>(s.rows, EDGE ? s.d + V - 1 : s.d, D.prof.sm_count, EACH, ROWS, period);
  return launch_rows(kernel, p.blocks, p.threads, smem, D.stream, 1, s, x, q, scale, p.group, period);
}

// Many rows at odd places.
template <typename T, int V, int EDGE>
int launch_edge(const DeviceSlot& D, const MapalQuantSite& s, const T* x, int8_t* q, float* scale) {
  const uint64_t span = s.d + V - 1;
  if (span <= 1024) return launch_flow<T, V, 8, 4, EDGE>(D, s, x, q, scale);
  if (span <= 8192) return launch_flow<T, V, 16, 2, EDGE>(D, s, x, q, scale);
  return launch_flow<T, V, 32, 1, EDGE>(D, s, x, q, scale);
}

template <typename T, int V>
int launch_quant(const DeviceSlot& D, const MapalQuantSite& s, const void* from, int8_t* q, float* scale) {
  const T* x = (const T*)from;
  // many: every thread of the device gets at least two turns of 32 elements
  const bool many = s.rows * s.d >= 64ull * kFlow * D.prof.sm_count;
  const uint64_t cap = 8ull * D.prof.sm_count;
  const unsigned blocks = (unsigned)(s.rows < cap ? s.rows : cap);
  if (many && s.d <= 1024) return launch_flow<T, V, 8, 4>(D, s, x, q, scale);
  if (many && s.d <= 8192) return launch_flow<T, V, 16, 2>(D, s, x, q, scale);
  if (many && s.d <= 16384) return launch_flow<T, V, 32, 1>(D, s, x, q, scale);
  if (s.d <= 8192)
    return launch_rows(quant_rows_kernel<T, V, 8>, blocks, s.d ? (int)((s.d + 255) / 256 * 32) : 32, 0, D.stream, 1, s, x, q,
                       scale);
  if (s.d <= 32768)
    return launch_rows(quant_rows_kernel<T, V, 32>, blocks, (int)((s.d + 1023) / 1024 * 32), 0, D.stream, 1, s, x, q, scale);
  return launch_rows(quant_rows_kernel<T, V, 0>, blocks, 1024, 0, D.stream, 1, s, x, q, scale);
}

// The widest access that x's rows, q's rows and a row's length allow.
template <typename T>
int by_width(const DeviceSlot& D, const MapalQuantSite& s, const void* x, int8_t* q, float* scale) {
  const int xw = align_of(x, s.ldx * sizeof(T), s.rows), qw = align_of(q, s.ldq, s.rows), dw = align_of(nullptr, s.d, 2);
  auto fits = [&](int v) { return xw >= v * (int)sizeof(T) && qw >= v && dw >= v; };
  constexpr int V = 16 / sizeof(T);
  if (fits(V)) return launch_quant<T, V>(D, s, x, q, scale);
  if constexpr (sizeof(T) == 2)
    if (fits(2)) return launch_quant<T, 2>(D, s, x, q, scale);
  if (s.d + V - 1 <= 16384 && s.rows * s.d >= kEdgeTurns * kFlow * D.prof.sm_count && aligned16(x) &&
      align_of(q, 0, 1) >= V) {
    if (s.rows > 1 && (s.ldx - s.ldq) % V != 0) return launch_edge<T, V, 2>(D, s, (const T*)x, q, scale);
    return launch_edge<T, V, 1>(D, s, (const T*)x, q, scale);
  }
  return launch_quant<T, 1>(D, s, x, q, scale);
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
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    const DeviceSlot& D = ctx->dev[0];
    MAPAL_TRY(site->dtype == MAPAL_DTYPE_F32   ? by_width<float>(D, *site, x, q, scale)
              : site->dtype == MAPAL_DTYPE_F16 ? by_width<__half>(D, *site, x, q, scale)
                                               : by_width<__nv_bfloat16>(D, *site, x, q, scale));
    return finish(ctx, 0, false);
  });
}

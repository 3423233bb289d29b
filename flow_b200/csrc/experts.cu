// experts.cu — tokens sorted by expert and back, with weights, and the
// gradients (mapal_gpu_expert_*). No counterpart in the reference; the rows'
// places follow its Index rule (a place outside the array traps index_oob).
//
// Slot t*k + j is token t's j-th expert. The sort is a counting sort: places
// are offsets[expert] + (earlier slots of that expert). Dispatch copies a
// token's row to its k places, combine adds k rows with weights; the gradient
// of either is the other's shape, so no sum ever needs an atomic.
#include <cooperative_groups.h>

#include "rows.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kTrapOob = 2;  // the trap flag's index_oob

// ---- sort --------------------------------------------------------------------------

constexpr int kMaxExperts = 1024;
constexpr int kSortWarps = 32;
constexpr int kSortThreads = kSortWarps * 32;
constexpr int kSortUnroll = 8;  // ids in flight for each lane

// One cluster sorts all slots, each warp a contiguous run of them in order.
// First walk: every warp counts its run's experts in its own row of shared
// counters (lanes with the same expert found with match.any, so a counter has
// one writer). Then counts become starting places: over warps in the block,
// over blocks through distributed shared memory, over experts by a block scan.
// Second walk: a slot's place is its expert's counter plus the lanes before it
// with the same expert. Slots keep their order within an expert, no atomics,
// no memory but the arrays.
__global__ void __launch_bounds__(kSortThreads) expert_sort_kernel(const int32_t* __restrict__ ids, uint32_t n, uint32_t E,
                                                                   uint32_t chunk, int32_t* __restrict__ offsets,
                                                                   int32_t* __restrict__ order,
                                                                   int32_t* __restrict__ pos, unsigned* trap) {
  extern __shared__ uint32_t sm[];
  uint32_t* cnt = sm;                      // [warp][E]
  uint32_t* total = sm + kSortWarps * E;   // [E]: this block's slots
  uint32_t* start = total + E;             // [E]: where this block's slots of an expert begin
  __shared__ uint32_t wsum[32];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t lt = (1u << lane) - 1;
  const uint64_t lo64 = (uint64_t)(rank * kSortWarps + warp) * chunk;
  const uint32_t lo = (uint32_t)(lo64 < n ? lo64 : n), hi = (uint32_t)(lo64 + chunk < n ? lo64 + chunk : n);
  uint32_t* mine = cnt + warp * E;

  for (uint32_t e = lane; e < E; e += 32) mine[e] = 0;
  __syncwarp();
  bool bad = false;
  for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kSortUnroll) {
    int32_t id[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const uint32_t i = i0 + u * 32 + lane;
      id[u] = i < hi ? __ldg(ids + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      if (i0 + u * 32 >= hi) break;
      const bool ok = (uint32_t)id[u] < E;
      bad |= !ok && id[u] != -1;
      const uint32_t same = __match_any_sync(0xffffffffu, ok ? id[u] : -1);
      if (ok && (same & lt) == 0) mine[id[u]] += __popc(same);
      __syncwarp();
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicMax(trap, kTrapOob);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < E; e += kSortThreads) {
    uint32_t run = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = cnt[w * E + e];
      cnt[w * E + e] = run;
      run += c;
    }
    total[e] = run;
  }
  cluster.sync();
  // E <= kSortThreads: one expert a thread
  uint32_t before = 0, all = 0;
  if (threadIdx.x < E)
    for (uint32_t r = 0; r < blocks; ++r) {
      const uint32_t c = *cluster.map_shared_rank(total + threadIdx.x, r);
      before += r < rank ? c : 0;
      all += c;
    }
  uint32_t incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  uint32_t base = 0;
  for (uint32_t w = 0; w < warp; ++w) base += wsum[w];
  if (threadIdx.x < E) {
    start[threadIdx.x] = base + incl - all + before;
    if (rank == 0) {
      offsets[threadIdx.x] = (int32_t)(base + incl - all);
      if (threadIdx.x == E - 1) offsets[E] = (int32_t)(base + incl);
    }
  }
  cluster.sync();  // `start` is written, and no block leaves while another reads its counts
  for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kSortUnroll) {
    int32_t id[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const uint32_t i = i0 + u * 32 + lane;
      id[u] = i < hi ? __ldg(ids + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      if (i0 + u * 32 >= hi) break;
      const uint32_t i = i0 + u * 32 + lane;
      const bool ok = (uint32_t)id[u] < E;
      const uint32_t same = __match_any_sync(0xffffffffu, ok ? id[u] : -1);
      int32_t p = -1;
      if (ok) {
        p = (int32_t)(start[id[u]] + mine[id[u]] + __popc(same & lt));
        if (order) order[p] = (int32_t)i;
      }
      __syncwarp();
      if (ok && (same & lt) == 0) mine[id[u]] += __popc(same);
      __syncwarp();
      if (i < hi) pos[i] = p;
    }
  }
}

// ---- rows --------------------------------------------------------------------------

constexpr int kThreads = 256;

// Token t's place for slot j, -1 for none; out of range raises the trap.
__device__ __forceinline__ int32_t place_of(const int32_t* pos, uint64_t slot, uint64_t rows, unsigned* trap) {
  const int32_t p = __ldg(pos + slot);
  if (p >= 0 && (uint64_t)p >= rows) {
    atomicMax(trap, kTrapOob);
    return -1;
  }
  return p;
}

// xs[pos[t, j]] = x[t] in units U of a row; one block a token.
template <typename U>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(const U* __restrict__ x, const float* __restrict__ scale,
                                                            const int32_t* __restrict__ pos, U* __restrict__ xs,
                                                            float* __restrict__ scale_out, uint64_t tokens, uint32_t k,
                                                            uint64_t units, uint64_t ldt, uint64_t ldr, uint64_t rows,
                                                            unsigned* trap) {
  for (uint64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    for (uint64_t i = threadIdx.x; i < units; i += kThreads) {
      const U v = x[t * ldt + i];
      for (uint32_t j = 0; j < k; ++j) {
        const int32_t p = place_of(pos, t * k + j, rows, trap);
        if (p >= 0) xs[(uint64_t)p * ldr + i] = v;
      }
    }
    if (scale)
      for (uint32_t j = threadIdx.x; j < k; j += kThreads) {
        const int32_t p = place_of(pos, t * k + j, rows, trap);
        if (p >= 0) scale_out[p] = scale[t];
      }
  }
}

// y[t] = sum_j w[t, j]*h[pos[t, j]]; one block a token.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) combine_kernel(const T* __restrict__ h, const float* __restrict__ w,
                                                           const int32_t* __restrict__ pos, T* __restrict__ y,
                                                           uint64_t tokens, uint32_t k, uint64_t d, uint64_t ldt,
                                                           uint64_t ldr, uint64_t rows, unsigned* trap) {
  for (uint64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    for (uint64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
      float acc[V] = {};
      for (uint32_t j = 0; j < k; ++j) {
        const int32_t p = place_of(pos, t * k + j, rows, trap);
        if (p < 0) continue;
        const float g = w ? __ldg(w + t * k + j) : 1.0f;
        float f[V];
        reinterpret_cast<const Pack<T, V>*>(h + (uint64_t)p * ldr + i)->get(f);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = __fmaf_rn(g, f[e], acc[e]);
      }
      Pack<T, V> o;
      o.set(acc);
      *reinterpret_cast<Pack<T, V>*>(y + t * ldt + i) = o;
    }
  }
}

// dh[p] = w*dy[t] and dw = <dy[t], h[p]>; one block a slot. An element of h is
// read by the thread that writes it in dh.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) combine_grad_kernel(const T* h, const float* __restrict__ w,
                                                                const int32_t* __restrict__ pos,
                                                                const T* __restrict__ dy, T* dh, float* __restrict__ dw,
                                                                uint64_t slots, uint32_t k, uint64_t d, uint64_t ldt,
                                                                uint64_t ldr, uint64_t rows, unsigned* trap) {
  __shared__ float red[2][32];
  int par = 0;
  for (uint64_t s = blockIdx.x; s < slots; s += gridDim.x, par ^= 1) {
    const int32_t p = place_of(pos, s, rows, trap);
    float dot = 0.0f;
    if (p >= 0) {
      const float g = w ? __ldg(w + s) : 1.0f;
      const T* dyr = dy + s / k * ldt;
      for (uint64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
        float a[V], b[V];
        reinterpret_cast<const Pack<T, V>*>(dyr + i)->get(a);
        reinterpret_cast<const Pack<T, V>*>(h + (uint64_t)p * ldr + i)->get(b);
        Pack<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          dot = __fmaf_rn(a[e], b[e], dot);
          a[e] *= g;
        }
        o.set(a);
        *reinterpret_cast<Pack<T, V>*>(dh + (uint64_t)p * ldr + i) = o;
      }
    }
    if (dw) {
      dot = block_sum(dot, red[par]);
      if (threadIdx.x == 0) dw[s] = dot;
    }
  }
}

// ---- host ------------------------------------------------------------------------------

int check_site(const MapalExpertSite* s, bool rows_arrays, bool bytes_too) {
  if (!s) return set_error(MAPAL_ERR_INVALID, "site is null");
  if (s->k == 0) return set_error(MAPAL_ERR_INVALID, "k is 0");
  if (s->experts == 0) return set_error(MAPAL_ERR_INVALID, "experts is 0");
  if (s->experts > kMaxExperts) return set_error(MAPAL_ERR_UNSUPPORTED, "more than 1024 experts");
  if (s->tokens > 0x7fffffffull / s->k) return set_error(MAPAL_ERR_INVALID, "tokens*k is 2^31 or more");
  if (!rows_arrays) return 0;
  const int es = dtype_bytes(s->dtype);
  if (es == 0 || (es == 1 && !bytes_too)) return set_error(MAPAL_ERR_INVALID, "the element type is not one this call takes");
  if (s->rows > 0x7fffffffull) return set_error(MAPAL_ERR_INVALID, "2^31 sorted rows or more");
  if (!rows_ok(s->tokens, s->d, s->ldt, es) || !rows_ok(s->rows, s->d, s->ldr, es))
    return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
  return 0;
}

bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

unsigned token_grid(uint64_t n, int sms) { return (unsigned)(n < 32ull * sms ? n : 32ull * sms); }

template <typename U>
void launch_dispatch(const DeviceSlot& D, const MapalExpertSite& s, const void* x, const float* scale, const int32_t* pos,
                     void* xs, float* scale_out) {
  const uint64_t es = dtype_bytes(s.dtype), u = sizeof(U);
  dispatch_kernel<U><<<token_grid(s.tokens, D.prof.sm_count), kThreads, 0, D.stream>>>(
      (const U*)x, scale, pos, (U*)xs, scale_out, s.tokens, s.k, s.d * es / u, s.ldt * es / u, s.ldr * es / u, s.rows,
      D.trap);
  count_launch();
}

// f(T, V) for the site's type and the widest access that the arrays allow.
template <typename F>
void by_type(const MapalExpertSite& s, int width, F&& f) {
  using std::integral_constant;
  if (s.dtype == MAPAL_DTYPE_F32) {
    if (width >= 16) return f(float{}, integral_constant<int, 4>{});
    return f(float{}, integral_constant<int, 1>{});
  }
  auto half = [&](auto t) {
    if (width >= 16) return f(t, integral_constant<int, 8>{});
    if (width >= 4) return f(t, integral_constant<int, 2>{});
    return f(t, integral_constant<int, 1>{});
  };
  if (s.dtype == MAPAL_DTYPE_F16) return half(__half{});
  return half(__nv_bfloat16{});
}

// The widest access that divides a row and at which both arrays' rows begin.
int row_width(const MapalExpertSite& s, const void* t, const void* t2, const void* r, const void* r2) {
  const uint64_t es = dtype_bytes(s.dtype);
  int w = align_of(t, s.ldt * es, s.tokens);
  for (const int o : {align_of(t2, s.ldt * es, s.tokens), align_of(r, s.ldr * es, s.rows),
                      align_of(r2, s.ldr * es, s.rows), align_of(nullptr, s.d * es, 2)})
    w = o < w ? o : w;
  return w;
}

}  // namespace

extern "C" int mapal_gpu_expert_sort(MapalGpuCtx* ctx, const MapalExpertSite* site, const int32_t* ids,
                                     int32_t* offsets, int32_t* order, int32_t* pos) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site, false, false));
    const uint64_t n = site->tokens * site->k;
    if (!offsets || (n && (!ids || !pos))) return set_error(MAPAL_ERR_INVALID, "null ids, offsets or pos");
    if (!aligned_to(ids, 4) || !aligned_to(offsets, 4) || !aligned_to(order, 4) || !aligned_to(pos, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    MAPAL_TRY(enter(ctx));
    DeviceSlot& D = ctx->dev[0];
    const uint32_t E = site->experts;
    const size_t smem = (size_t)(kSortWarps + 2) * E * sizeof(uint32_t);
    static std::atomic<uint64_t> done{0};
    MAPAL_TRY(ensure_smem_attr(done, (const void*)expert_sort_kernel, D.device,
                               (size_t)(kSortWarps + 2) * kMaxExperts * sizeof(uint32_t), "expert_sort shared memory"));
    const unsigned blocks = n <= 4096 ? 1 : n <= 8192 ? 2 : n <= 16384 ? 4 : 8;
    const uint64_t warps = (uint64_t)blocks * kSortWarps;
    const uint32_t chunk = (uint32_t)(((n + warps - 1) / warps + 31) / 32 * 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = D.stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    MAPAL_CUDA(cudaLaunchKernelEx(&cfg, expert_sort_kernel, ids, (uint32_t)n, E, chunk, offsets, order, pos, D.trap));
    count_launch();
    return finish(ctx, 0, true);
  });
}

extern "C" int mapal_gpu_expert_dispatch(MapalGpuCtx* ctx, const MapalExpertSite* site, const void* x,
                                         const float* scale, const int32_t* pos, void* xs, float* scale_out) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site, true, true));
    if (site->tokens == 0) return 0;
    if (!pos || (site->d && (!x || (!xs && site->rows)))) return set_error(MAPAL_ERR_INVALID, "null x, pos or xs");
    if (!scale != !scale_out) return set_error(MAPAL_ERR_INVALID, "scale and scale_out come together");
    const int es = dtype_bytes(site->dtype);
    if (!aligned_to(x, es) || !aligned_to(xs, es) || !aligned_to(pos, 4) || !aligned_to(scale, 4) ||
        !aligned_to(scale_out, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    MAPAL_TRY(enter(ctx));
    DeviceSlot& D = ctx->dev[0];
    switch (row_width(*site, x, x, xs, xs)) {
      case 16: launch_dispatch<uint4>(D, *site, x, scale, pos, xs, scale_out); break;
      case 8: launch_dispatch<uint2>(D, *site, x, scale, pos, xs, scale_out); break;
      case 4: launch_dispatch<uint32_t>(D, *site, x, scale, pos, xs, scale_out); break;
      case 2: launch_dispatch<uint16_t>(D, *site, x, scale, pos, xs, scale_out); break;
      default: launch_dispatch<uint8_t>(D, *site, x, scale, pos, xs, scale_out); break;
    }
    return finish(ctx, 0, true);
  });
}

static int combine_rows(MapalGpuCtx* ctx, const MapalExpertSite* site, const void* h, const float* w,
                        const int32_t* pos, void* y) {
  MAPAL_TRY(check_site(site, true, false));
  if (site->tokens == 0 || site->d == 0) return 0;
  if (!pos || !y || (!h && site->rows)) return set_error(MAPAL_ERR_INVALID, "null rows or pos");
  const int es = dtype_bytes(site->dtype);
  if (!aligned_to(h, es) || !aligned_to(y, es) || !aligned_to(pos, 4) || !aligned_to(w, 4))
    return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
  MAPAL_TRY(enter(ctx));
  DeviceSlot& D = ctx->dev[0];
  const MapalExpertSite& s = *site;
  by_type(s, row_width(s, y, y, h, h), [&](auto t, auto v) {
    using T = decltype(t);
    combine_kernel<T, v.value><<<token_grid(s.tokens, D.prof.sm_count), kThreads, 0, D.stream>>>(
        (const T*)h, w, pos, (T*)y, s.tokens, s.k, s.d, s.ldt, s.ldr, s.rows, D.trap);
    count_launch();
  });
  return finish(ctx, 0, true);
}

extern "C" int mapal_gpu_expert_combine(MapalGpuCtx* ctx, const MapalExpertSite* site, const void* h, const float* w,
                                        const int32_t* pos, void* y) {
  return guarded([&]() -> int { return combine_rows(ctx, site, h, w, pos, y); });
}

extern "C" int mapal_gpu_expert_dispatch_grad(MapalGpuCtx* ctx, const MapalExpertSite* site, const void* dxs,
                                              const int32_t* pos, void* dx) {
  return guarded([&]() -> int { return combine_rows(ctx, site, dxs, nullptr, pos, dx); });
}

extern "C" int mapal_gpu_expert_combine_grad(MapalGpuCtx* ctx, const MapalExpertSite* site, const void* h,
                                             const float* w, const int32_t* pos, const void* dy, void* dh, float* dw) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site, true, false));
    if (site->tokens == 0) return 0;
    if (!pos || (site->d && (!dy || (site->rows && (!h || !dh)))))
      return set_error(MAPAL_ERR_INVALID, "null h, pos, dy or dh");
    const int es = dtype_bytes(site->dtype);
    if (!aligned_to(h, es) || !aligned_to(dy, es) || !aligned_to(dh, es) || !aligned_to(pos, 4) || !aligned_to(w, 4) ||
        !aligned_to(dw, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    MAPAL_TRY(enter(ctx));
    DeviceSlot& D = ctx->dev[0];
    const MapalExpertSite& s = *site;
    by_type(s, row_width(s, dy, dy, h, dh), [&](auto t, auto v) {
      using T = decltype(t);
      const uint64_t slots = s.tokens * s.k;
      combine_grad_kernel<T, v.value><<<token_grid(slots, D.prof.sm_count), kThreads, 0, D.stream>>>(
          (const T*)h, w, pos, (const T*)dy, (T*)dh, dw, slots, s.k, s.d, s.ldt, s.ldr, s.rows, D.trap);
      count_launch();
    });
    return finish(ctx, 0, true);
  });
}

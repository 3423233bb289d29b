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
constexpr int kSortWarps = 32;  // at most, in a block
constexpr int kSortThreads = kSortWarps * 32;
constexpr uint32_t kSortBlocks = 8;  // at most, in the cluster
constexpr int kThreads = 256;
constexpr int kSortUnroll = 8;  // ids in flight for each lane

// Lanes (of those with ok) that have the same id, which has `bits` bits: a
// ballot for each bit. match.any answers the same question some eight times
// slower when the ids differ (2^20 slots of 64 experts: 254 us with it).
__device__ __forceinline__ uint32_t same_id(int32_t id, bool ok, int bits) {
  uint32_t same = __ballot_sync(0xffffffffu, ok);
  for (int b0 = 0; b0 < bits; b0 += 4)
#pragma unroll
    for (int b = b0; b < b0 + 4; ++b) {  // a bit that no id has changes nothing
      const bool one = (id >> b) & 1;
      const uint32_t ones = __ballot_sync(0xffffffffu, ok && one);
      same &= one ? ones : ~ones;
    }
  return same;
}

// One cluster sorts all slots, each warp a contiguous run of them in order.
// First walk: every warp counts its run's experts in its own row of shared
// counters (lanes with the same expert are found with ballots, so a counter has
// one writer). Then counts become starting places: over warps in the block,
// over blocks through distributed shared memory, over experts by a block scan.
// Second walk: a slot's place is its expert's counter plus the lanes before it
// with the same expert. Slots keep their order within an expert, no atomics,
// no memory but the arrays.
__global__ void __launch_bounds__(kSortThreads)
    expert_sort_kernel(const int32_t* __restrict__ ids, uint32_t n, uint32_t E, uint32_t chunk,
                       int32_t* __restrict__ offsets, int32_t* __restrict__ order, int32_t* __restrict__ pos,
                       unsigned* trap) {
  extern __shared__ uint32_t sm[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t* cnt = sm;                 // [warp][E]
  uint32_t* total = sm + warps * E;   // [E]: this block's slots
  uint32_t* start = total + E;        // [E]: where this block's slots of an expert begin
  __shared__ uint32_t wsum[32];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const uint32_t lt = (1u << lane) - 1;
  const int bits = 32 - __clz(E - 1);
  const uint64_t lo64 = (uint64_t)(rank * warps + warp) * chunk;
  const uint32_t lo = (uint32_t)(lo64 < n ? lo64 : n), hi = (uint32_t)(lo64 + chunk < n ? lo64 + chunk : n);
  uint32_t* mine = cnt + warp * E;

  auto load = [&](int32_t (&id)[kSortUnroll], uint32_t i0) {
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const uint32_t i = i0 + u * 32 + lane;
      id[u] = i < hi ? __ldg(ids + i) : -1;
    }
  };
  for (uint32_t e = lane; e < E; e += 32) mine[e] = 0;
  grid_wait();
  grid_go();
  int32_t id[kSortUnroll];
  load(id, lo);
  __syncwarp();
  bool bad = false;
  for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kSortUnroll) {
    if (i0 != lo) load(id, i0);
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      if (i0 + u * 32 >= hi) break;
      const bool ok = (uint32_t)id[u] < E;
      bad |= !ok && id[u] != -1;
      const uint32_t same = same_id(id[u], ok, bits);
      if (ok && (same & lt) == 0) mine[id[u]] += __popc(same);
      __syncwarp();
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicMax(trap, kTrapOob);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < E; e += blockDim.x) {
    uint32_t run = 0;
    for (uint32_t w0 = 0; w0 < warps; w0 += 8) {
      uint32_t c[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) c[w] = w0 + w < warps ? cnt[(w0 + w) * E + e] : 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (w0 + w < warps) cnt[(w0 + w) * E + e] = run;
        run += c[w];
      }
    }
    total[e] = run;
  }
  if (blocks > 1)
    cluster.sync();
  else
    __syncthreads();
  // blocks of blockDim.x experts in turn, one a thread
  uint32_t done = 0;
  for (uint32_t e0 = 0; e0 < E; e0 += blockDim.x) {
    const uint32_t e = e0 + threadIdx.x;
    uint32_t before = 0, all = 0;
    if (e < E) {
      uint32_t c[kSortBlocks];
#pragma unroll
      for (uint32_t r = 0; r < kSortBlocks; ++r)
        c[r] = r >= blocks ? 0 : blocks > 1 ? *cluster.map_shared_rank(total + e, r) : total[e];
#pragma unroll
      for (uint32_t r = 0; r < kSortBlocks; ++r) {
        before += r < rank ? c[r] : 0;
        all += c[r];
      }
    }
    uint32_t incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    const uint32_t part = lane < warps ? wsum[lane] : 0;
    const uint32_t base = done + __reduce_add_sync(0xffffffffu, lane < warp ? part : 0);
    done += __reduce_add_sync(0xffffffffu, part);
    if (e < E) {
      start[e] = base + incl - all + before;
      if (rank == 0) offsets[e] = (int32_t)(base + incl - all);
    }
    __syncthreads();
  }
  if (rank == 0 && threadIdx.x == 0) offsets[E] = (int32_t)done;
  for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kSortUnroll) {
    if (chunk > 32 * kSortUnroll) load(id, i0);  // a shorter run is still held
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      if (i0 + u * 32 >= hi) break;
      const uint32_t i = i0 + u * 32 + lane;
      const bool ok = (uint32_t)id[u] < E;
      const uint32_t same = same_id(id[u], ok, bits);
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
  if (blocks > 1) cluster.sync();  // no block leaves while another reads its counts
}

// ---- rows --------------------------------------------------------------------------
//
// Bound by HBM: dispatch reads a token's row once and writes k, combine reads k
// and writes one. A block takes a piece of a token's row (a few accesses a
// thread), so that even a few tokens spread over the device, and each thread
// has all of its loads in flight at once.

constexpr int kRowThreads = 128;
constexpr int kAtOnce = 4;  // slots of a token whose rows are in flight together

// Slot's place, -1 for none; out of range raises the trap.
__device__ __forceinline__ int32_t place_of(const int32_t* pos, uint64_t slot, uint64_t rows, unsigned* trap) {
  const int32_t p = __ldg(pos + slot);
  if (p >= 0 && (uint64_t)p >= rows) {
    atomicMax(trap, kTrapOob);
    return -1;
  }
  return p;
}

// A row in pieces of `piece` accesses; item = token * pieces + piece.
struct Pieces {
  uint64_t items;
  uint32_t pieces;
};

// xs[pos[t, j]] = x[t] in units U of a row, NV units a thread.
template <typename U, int NV>
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(const U* __restrict__ x, const float* __restrict__ scale,
                                                               const int32_t* __restrict__ pos, U* __restrict__ xs,
                                                               float* __restrict__ scale_out, Pieces Q, uint32_t k,
                                                               uint64_t units, uint64_t ldt, uint64_t ldr,
                                                               uint64_t rows, unsigned* trap) {
  grid_wait();
  grid_go();
  for (uint64_t item = blockIdx.x; item < Q.items; item += gridDim.x) {
    const uint64_t t = item / Q.pieces;
    const uint32_t piece = (uint32_t)(item % Q.pieces);
    const uint64_t i0 = (uint64_t)piece * (kRowThreads * NV) + threadIdx.x;
    U v[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (i0 + u * kRowThreads < units) v[u] = x[t * ldt + i0 + u * kRowThreads];
    for (uint32_t j = 0; j < k; ++j) {
      const int32_t p = place_of(pos, t * k + j, rows, trap);
      if (p < 0) continue;
      U* to = xs + (uint64_t)p * ldr + i0;
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (i0 + u * kRowThreads < units) to[u * kRowThreads] = v[u];
      if (scale && piece == 0 && threadIdx.x == 0) scale_out[p] = scale[t];
    }
  }
}

// y[t] = sum_j w[t, j]*h[pos[t, j]], NV packs a thread.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(const T* __restrict__ h, const float* __restrict__ w,
                                                              const int32_t* __restrict__ pos, T* __restrict__ y,
                                                              Pieces Q, uint32_t k, uint64_t d, uint64_t ldt,
                                                              uint64_t ldr, uint64_t rows, unsigned* trap) {
  using P = Pack<T, V>;
  grid_wait();
  grid_go();
  for (uint64_t item = blockIdx.x; item < Q.items; item += gridDim.x) {
    const uint64_t t = item / Q.pieces;
    const uint64_t i0 = ((item % Q.pieces) * (kRowThreads * NV) + threadIdx.x) * V;
    float acc[NV][V] = {};
    for (uint32_t j0 = 0; j0 < k; j0 += kAtOnce) {
      P v[kAtOnce][NV];
      float g[kAtOnce];
      bool on[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const uint64_t slot = t * k + j0 + u;
        const int32_t p = j0 + u < k ? place_of(pos, slot, rows, trap) : -1;
        on[u] = p >= 0;
        g[u] = on[u] && w ? __ldg(w + slot) : 1.0f;
        const T* from = h + (uint64_t)(on[u] ? p : 0) * ldr + i0;
#pragma unroll
        for (int c = 0; c < NV; ++c)
          if (on[u] && i0 + c * (kRowThreads * V) < d) v[u][c] = ld_once(reinterpret_cast<const P*>(from + c * (kRowThreads * V)));
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (on[u]) {
#pragma unroll
          for (int c = 0; c < NV; ++c) {
            float f[V];
            v[u][c].get(f);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[c][e] = __fmaf_rn(g[u], f[e], acc[c][e]);
          }
        }
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      P o;
      o.set(acc[c]);
      if (i0 + c * (kRowThreads * V) < d) st_once(reinterpret_cast<P*>(y + t * ldt + i0 + c * (kRowThreads * V)), o);
    }
  }
}

// dh[p] = w*dy[t] and dw = <dy[t], h[p]> for SLOTS slots of a token at once,
// over which dy is read once; a block owns whole rows, so dw needs no atomics.
// An element of h is read by the thread that writes it in dh.
template <typename T, int V, int SLOTS>
__global__ void __launch_bounds__(kThreads) combine_grad_kernel(const T* h, const float* __restrict__ w,
                                                                const int32_t* __restrict__ pos,
                                                                const T* __restrict__ dy, T* dh, float* __restrict__ dw,
                                                                uint64_t items, uint32_t k, uint64_t d, uint64_t ldt,
                                                                uint64_t ldr, uint64_t rows, unsigned* trap) {
  using P = Pack<T, V>;
  __shared__ float red[2][SLOTS][kThreads / 32];
  const uint32_t turns = (k + SLOTS - 1) / SLOTS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int par = 0;
  grid_wait();
  grid_go();
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x, par ^= 1) {
    const uint64_t t = item / turns;
    const uint32_t j0 = (uint32_t)(item % turns) * SLOTS;
    float dot[SLOTS], g[SLOTS];
    uint64_t at[SLOTS];
    bool on[SLOTS];
#pragma unroll
    for (int u = 0; u < SLOTS; ++u) {
      const uint64_t slot = t * k + j0 + u;
      const int32_t p = j0 + u < k ? place_of(pos, slot, rows, trap) : -1;
      on[u] = p >= 0;
      g[u] = on[u] && w ? __ldg(w + slot) : 1.0f;
      at[u] = (uint64_t)(on[u] ? p : 0) * ldr;
      dot[u] = 0.0f;
    }
    const T* dyr = dy + t * ldt;
    // all loads of a turn before its stores: dh may be h, so the compiler keeps their order
    constexpr int NV = sizeof(P) == 16 ? 1 : 4;
    const uint64_t step = blockDim.x * V;
    for (uint64_t i0 = threadIdx.x * V; i0 < d; i0 += step * NV) {
      P a[NV], b[SLOTS][NV];
#pragma unroll
      for (int c = 0; c < NV; ++c)
        if (i0 + c * step < d) a[c] = *reinterpret_cast<const P*>(dyr + i0 + c * step);
#pragma unroll
      for (int u = 0; u < SLOTS; ++u)
        if (on[u]) {
#pragma unroll
          for (int c = 0; c < NV; ++c)
            if (i0 + c * step < d) b[u][c] = ld_once(reinterpret_cast<const P*>(h + at[u] + i0 + c * step));
        }
#pragma unroll
      for (int u = 0; u < SLOTS; ++u)
        if (on[u]) {
#pragma unroll
          for (int c = 0; c < NV; ++c)
            if (i0 + c * step < d) {
              float fa[V], fb[V];
              a[c].get(fa);
              b[u][c].get(fb);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                dot[u] = __fmaf_rn(fa[e], fb[e], dot[u]);
                fb[e] = fa[e] * g[u];
              }
              P o;
              o.set(fb);
              st_once(reinterpret_cast<P*>(dh + at[u] + i0 + c * step), o);
            }
        }
    }
    if (dw) {
#pragma unroll
      for (int u = 0; u < SLOTS; ++u) {
        dot[u] = warp_sum(dot[u]);
        if (lane == 0) red[par][u][warp] = dot[u];
      }
      __syncthreads();
      if (threadIdx.x < SLOTS && j0 + threadIdx.x < k) {
        float s = 0.0f;
        for (int q = 0; q < warps; ++q) s += red[par][threadIdx.x][q];
        dw[t * k + j0 + threadIdx.x] = s;
      }
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
  if (s->d > 0x7fffffffull) return set_error(MAPAL_ERR_INVALID, "rows of 2^31 elements or more");
  if (s->rows > 0x7fffffffull) return set_error(MAPAL_ERR_INVALID, "2^31 sorted rows or more");
  if (!rows_ok(s->tokens, s->d, s->ldt, es) || !rows_ok(s->rows, s->d, s->ldr, es))
    return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
  return 0;
}

bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

constexpr uint64_t kMostBlocks = 1u << 20;  // what lies beyond is walked

// `accesses` of a row, NV a thread.
Pieces pieces_of(uint64_t tokens, uint64_t accesses, int nv) {
  Pieces q;
  const uint64_t one = (uint64_t)kRowThreads * nv;
  q.pieces = (uint32_t)((accesses + one - 1) / one);
  if (q.pieces == 0) q.pieces = 1;
  q.items = tokens * q.pieces;
  return q;
}

template <typename U>
int launch_dispatch(const DeviceSlot& D, const MapalExpertSite& s, const void* x, const float* scale, const int32_t* pos,
                     void* xs, float* scale_out) {
  const uint64_t es = dtype_bytes(s.dtype), u = sizeof(U);
  constexpr int NV = sizeof(U) == 16 ? 2 : 4;
  const Pieces q = pieces_of(s.tokens, s.d * es / u, NV);
  return launch_rows(dispatch_kernel<U, NV>, (unsigned)(q.items < kMostBlocks ? q.items : kMostBlocks), kRowThreads, 0,
                     D.stream, 1, (const U*)x, scale, pos, (U*)xs, scale_out, q, s.k, s.d * es / u, s.ldt * es / u,
                     s.ldr * es / u, s.rows, D.trap);
}

// f(T, V) for the site's type and the widest access that the arrays allow.
template <typename F>
int by_type(const MapalExpertSite& s, int width, F&& f) {
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
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    const uint32_t E = site->experts;
    static std::atomic<uint64_t> done{0};
    MAPAL_TRY(ensure_smem_attr(done, (const void*)expert_sort_kernel, D.device,
                               (size_t)(kSortWarps + 2) * kMaxExperts * sizeof(uint32_t), "expert_sort shared memory"));
    // About 64 slots a warp: a few warps of one block sort a generated batch,
    // 8 blocks more (1024 slots of 64 experts 4 us either way, 4096: 8 and 5).
    const uint64_t want = (n + 63) / 64;
    const unsigned blocks = n <= 1024 ? 1 : kSortBlocks;
    const uint64_t share = (want + blocks - 1) / blocks;
    const uint64_t least = E / 64 < 4 ? 4 : E / 64;  // an expert is a thread's when places are counted
    const uint32_t warps = (uint32_t)(share > kSortWarps ? kSortWarps : share > least ? share : least);
    const uint64_t all = (uint64_t)blocks * warps;
    const uint32_t chunk = (uint32_t)(((n + all - 1) / all + 31) / 32 * 32);
    const size_t smem = (size_t)(warps + 2) * E * sizeof(uint32_t);
    MAPAL_TRY(launch_rows(expert_sort_kernel, blocks, (int)warps * 32, smem, D.stream, blocks, ids, (uint32_t)n, E, chunk,
                          offsets, order, pos, D.trap));
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
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    switch (row_width(*site, x, x, xs, xs)) {
      case 16: MAPAL_TRY(launch_dispatch<uint4>(D, *site, x, scale, pos, xs, scale_out)); break;
      case 8: MAPAL_TRY(launch_dispatch<uint2>(D, *site, x, scale, pos, xs, scale_out)); break;
      case 4: MAPAL_TRY(launch_dispatch<uint32_t>(D, *site, x, scale, pos, xs, scale_out)); break;
      case 2: MAPAL_TRY(launch_dispatch<uint16_t>(D, *site, x, scale, pos, xs, scale_out)); break;
      default: MAPAL_TRY(launch_dispatch<uint8_t>(D, *site, x, scale, pos, xs, scale_out)); break;
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
  const OnDevice on(ctx);
  MAPAL_TRY(on.rc);
  DeviceSlot& D = ctx->dev[0];
  const MapalExpertSite& s = *site;
  MAPAL_TRY(by_type(s, row_width(s, y, y, h, h), [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = v.value, NV = V * sizeof(T) == 16 ? 1 : 4;
    const Pieces q = pieces_of(s.tokens, s.d / V, NV);
    return launch_rows(combine_kernel<T, V, NV>, (unsigned)(q.items < kMostBlocks ? q.items : kMostBlocks), kRowThreads, 0,
                       D.stream, 1, (const T*)h, w, pos, (T*)y, q, s.k, s.d, s.ldt, s.ldr, s.rows, D.trap);
  }));
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
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    const MapalExpertSite& s = *site;
    MAPAL_TRY(by_type(s, row_width(s, dy, dy, h, dh), [&](auto t, auto v) {
      using T = decltype(t);
      constexpr int V = v.value;
      const uint64_t wide = (s.d / V + 31) / 32 * 32;
      const unsigned threads = wide < 32 ? 32 : wide < kThreads ? (unsigned)wide : kThreads;
      // tokens that do not fill the device go slot by slot
      const bool few = s.tokens < 8ull * D.prof.sm_count;
      const uint64_t items = s.tokens * (few ? s.k : (s.k + kAtOnce - 1) / kAtOnce);
      auto kernel = few ? combine_grad_kernel<T, V, 1> : combine_grad_kernel<T, V, kAtOnce>;
      return launch_rows(kernel, (unsigned)(items < kMostBlocks ? items : kMostBlocks), (int)threads, 0, D.stream, 1,
                         (const T*)h, w, pos, (const T*)dy, (T*)dh, dw, items, s.k, s.d, s.ldt, s.ldr, s.rows, D.trap);
    }));
    return finish(ctx, 0, true);
  });
}

// norm.cu — layer norm over rows, forward and backward (mapal_gpu_layer_norm,
// mapal_gpu_layer_norm_grad). No counterpart in the reference.
//
// Forward: mu = mean(x), r = 1/sqrt(mean((x - mu)^2) + eps), y = (x - mu)*r*w + b.
// Backward, with h = (x - mu)*r and g = dy*w:
//   dx = r*(g - mean(g) - h*mean(g*h)), dw = sum_rows dy*h, db = sum_rows dy.
#include "f32x2.cuh"
#include "rowflow.cuh"

namespace {

constexpr int kThreads = 256;  // of the kernels for long rows
constexpr int kMostFlow = 8192;  // elements of the longest row of the kernels for many rows

// V weights of type TW as floats; `none` where there are no weights.
template <typename TW, int V>
__device__ __forceinline__ void weights(const void* w, int64_t i, float none, float (&out)[V]) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = none;
  } else {
    constexpr int U = V * sizeof(TW) > 16 ? 16 / sizeof(TW) : V;  // elements of an access
#pragma unroll
    for (int u = 0; u < V; u += U) {
      float f[U];
      reinterpret_cast<const Pack<TW, U>*>(static_cast<const TW*>(w) + i + u)->get(f);
#pragma unroll
      for (int e = 0; e < U; ++e) out[u + e] = f[e];
    }
  }
}

// The same for columns i to i + V - 1 of d, which need not be aligned or all
// exist; zeros for those that do not.
template <typename TW, int V>
__device__ __forceinline__ void weights_at(const void* w, int i, int d, float none, float (&out)[V]) {
  if (i >= 0 && i + V <= d && i % V == 0) {
    weights<TW, V>(w, i, none, out);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      out[e] = i + e < 0 || i + e >= d ? 0.0f : w ? to_f32(__ldg(static_cast<const TW*>(w) + i + e)) : none;
  }
}

__device__ __forceinline__ float inv_std(float var, float eps) { return __fdiv_rn(1.0f, __fsqrt_rn(var + eps)); }


// ---- few rows ------------------------------------------------------------------------
//
// Forward: a row lives, packed as it was read, in the registers of a group of
// warps, EACH elements a thread, so it is read once and both sums run over
// registers. 8 elements a thread spread a row's loads and sums as wide as they
// go; rows of more than 8192 elements take 16 or 32 a thread.

template <typename T, typename TW, int V, int EACH>
__global__ void __launch_bounds__(1024)
    norm_held_kernel(const MapalNormSite S, const T* x, const void* __restrict__ w, const void* __restrict__ b, T* y,
                     float* __restrict__ mean, float* __restrict__ rstd, int group) {
  using P = Pack<T, V>;
  constexpr int NV = EACH / V;
  __shared__ float red[32][2][32];  // at most 32 groups
  const Group<false> G(group);
  grid_wait();
  grid_go();
  const uint64_t stride = (uint64_t)gridDim.x * (blockDim.x / group);
  const int d = (int)S.d;
  const float n = (float)d;
  for (uint64_t r = (uint64_t)blockIdx.x * (blockDim.x / group) + G.id; r < S.rows; r += stride) {
    const T* xr = x + r * S.ldx;
    P v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * group + G.tid) * V;
      if (i < d)
        v[j] = ld_once(reinterpret_cast<const P*>(xr + i));
      else
        v[j].clear();
    }
    // with few elements a thread the weights are asked for along with the row
    constexpr bool kAhead = EACH == 8 && sizeof(P) == 16;
    float fw[kAhead ? 8 : 1], fb[kAhead ? 8 : 1];
    if constexpr (kAhead) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (j * group + G.tid) * V;
        float pw[V] = {}, pb[V] = {};
        if (i < d) {
          weights<TW, V>(w, i, 1.0f, pw);
          weights<TW, V>(b, i, 0.0f, pb);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          fw[j * V + e] = pw[e];
          fb[j * V + e] = pb[e];
        }
      }
    }
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[V];
      v[j].get(f);
#pragma unroll
      for (int e = 0; e < V; ++e) s += f[e];
    }
    const float mu = __fdiv_rn(G.sum(s, red[G.id][0]), n);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if ((j * group + G.tid) * V < d) {
        if constexpr (EACH > 8) v[j].forget();
        float f[V];
        v[j].get(f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float c = f[e] - mu;
          q = __fmaf_rn(c, c, q);
        }
      }
    const float rs = inv_std(__fdiv_rn(G.sum(q, red[G.id][1]), n), S.eps);
    T* yr = y + r * S.ldy;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * group + G.tid) * V;
      if (i < d) {
        if constexpr (EACH > 8) v[j].forget();
        float f[V], pw[V], pb[V];
        v[j].get(f);
        if constexpr (kAhead) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            pw[e] = fw[j * V + e];
            pb[e] = fb[j * V + e];
          }
        } else {
          weights<TW, V>(w, i, 1.0f, pw);
          weights<TW, V>(b, i, 0.0f, pb);
        }
        P o;
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = __fmaf_rn((f[e] - mu) * rs, pw[e], pb[e]);
        o.set(f);
        st_once(reinterpret_cast<P*>(yr + i), o);
      }
      if constexpr (EACH > 8) asm volatile("" ::: "memory");  // keeps the weights' loads from piling up in registers
    }
    if (G.tid == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

// ---- many rows of up to 8192 elements ------------------------------------------------
//
// A group of threads takes ROWS rows at a time through the ring, EACH columns a
// thread, and keeps its columns' weights (and, in the gradient, their sums over
// rows) in registers from row to row. What is left is instructions, so the
// arithmetic is on packed pairs and the sums of ROWS rows share their shuffles
// and barrier.

__device__ __forceinline__ float f2_sum(f2 v) { return f2_lo(v) + f2_hi(v); }

template <typename T, typename TW, int V, int EACH, int ROWS, bool SUB, int EDGE>
__global__ void __launch_bounds__(kFlow, 1)
    norm_flow_kernel(const MapalNormSite S, const T* x, const void* __restrict__ w, const void* __restrict__ b, T* y,
                     float* __restrict__ mean, float* __restrict__ rstd, int group, uint32_t period) {
  using R = std::conditional_t<EDGE != 0, EdgeRing<T, EACH, ROWS, 1, SUB, EDGE == 2>, Ring<T, V, EACH, ROWS, 1>>;
  using P = Pack<T, V>;
  constexpr int NV = EACH / V;
  __shared__ float sets[kMostGroups][2][4][16];
  extern __shared__ __align__(16) uint8_t dyn[];
  const Group<SUB> G(group);
  R ring(dyn, G);
  auto* red = sets[SUB || group == 32 ? 0 : G.id];
  const Turns<SUB, EDGE, ROWS> mine(G, period, S.rows);
  uint64_t rows = mine.rows, ldx = mine.stride(S.ldx), ldy = mine.stride(S.ldy);
  uint64_t r = mine.first;
  const int d = (int)S.d, shift = mine.template shift<T>(S.ldy), shift_x = mine.template shift<T>(S.ldx);
  const std::conditional_t<EDGE != 0, Input<V, NV>, Whole> in(group, G.tid, d, shift_x, shift);
  const std::conditional_t<EDGE != 0, Mine<V, NV>, Whole> part(group, G.tid, shift, d + shift);
  const std::conditional_t<EDGE != 0, Masks<P, V, NV>, Whole> keep(part);
  x = mine.at(x, S.ldx) - shift_x + (G.tid - in.back) * V;
  y = mine.at(y, S.ldy) - shift + G.tid * V;
  mean = mine.at(mean, 1);
  rstd = mine.at(rstd, 1);
  if constexpr (EDGE != 0) {
    pin(x), pin(y);
    pin(rows), pin(ldx), pin(ldy);
  }
  const float n = (float)d;
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
  f2 fw[EACH / 2], fb[EACH / 2];
  {
    float a[EACH], c[EACH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * group + G.tid) * V;
      float pa[V] = {}, pc[V] = {};
      if constexpr (EDGE != 0) {
        weights_at<TW, V>(w, i - shift, d, 1.0f, pa);
        weights_at<TW, V>(b, i - shift, d, 0.0f, pc);
      } else if (i < d) {
        weights<TW, V>(w, i, 1.0f, pa);
        weights<TW, V>(b, i, 0.0f, pc);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        a[j * V + e] = pa[e];
        c[j * V + e] = pc[e];
      }
    }
#pragma unroll
    for (int u = 0; u < EACH / 2; ++u) {
      fw[u] = f2_pack(a[2 * u], a[2 * u + 1]);
      fb[u] = f2_pack(c[2 * u], c[2 * u + 1]);
    }
  }
  for (; r < rows; r += mine.step) {
    ring.wait();
    f2 v[ROWS][EACH / 2];
    float s[ROWS], q[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      float f[EACH];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        P p;
        if constexpr (EDGE != 0) {
          p = ring.take(k * NV + j, in.by);
          keep(p, j);
        } else if ((j * group + G.tid) * V < d && r + k < rows) {
          p = ring.take(k * NV + j);
        } else {
          p.clear();
        }
        float g[V];
        p.get(g);
#pragma unroll
        for (int e = 0; e < V; ++e) f[j * V + e] = g[e];
      }
      f2 t = f2_splat(0.0f);
#pragma unroll
      for (int u = 0; u < EACH / 2; ++u) {
        v[k][u] = f2_pack(f[2 * u], f[2 * u + 1]);
        t = f2_add(t, v[k][u]);
      }
      s[k] = f2_sum(t);
    }
    G.sums(s, red[0]);
    if constexpr (EDGE != 0) ring.taken();
    start(ring.stage, r + R::kStages * mine.step);  // this turn's slots have been read
    ring.next_stage();
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      s[k] = __fdiv_rn(s[k], n);
      const f2 m = f2_splat(-s[k]);
#pragma unroll
      for (int u = 0; u < EACH / 2; ++u) v[k][u] = f2_add(v[k][u], m);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (EDGE != 0) {
          const uint32_t own = part.at(j);
          if (own != part.kAll)
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              f2& u = v[k][(j * V + e) / 2];
              u = f2_pack(own & (1u << e) ? f2_lo(u) : 0.0f, own & (2u << e) ? f2_hi(u) : 0.0f);
            }
        } else if ((j * group + G.tid) * V >= d) {  // no elements here
          if constexpr (V > 1) {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) v[k][j * (V / 2) + e] = f2_splat(0.0f);
          } else {
            v[k][j / 2] = j % 2 ? f2_pack(f2_lo(v[k][j / 2]), 0.0f) : f2_pack(0.0f, f2_hi(v[k][j / 2]));
          }
        }
      }
      f2 t = f2_splat(0.0f);
#pragma unroll
      for (int u = 0; u < EACH / 2; ++u) t = f2_fma(v[k][u], v[k][u], t);
      q[k] = f2_sum(t);
    }
    G.sums(q, red[1]);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const float rs = inv_std(__fdiv_rn(q[k], n), S.eps);
      if (r + k >= rows) break;
      const f2 m = f2_splat(rs);
      float f[EACH];
#pragma unroll
      for (int u = 0; u < EACH / 2; ++u) {
        const f2 o = f2_fma(f2_mul(v[k][u], m), fw[u], fb[u]);
        f[2 * u] = f2_lo(o);
        f[2 * u + 1] = f2_hi(o);
      }
      T* to = y + (r + k) * ldy;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float g[V];
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = f[j * V + e];
        P p;
        p.set(g);
        if constexpr (EDGE != 0) {
          if (part.at(j) == part.kAll)
            st_once(reinterpret_cast<P*>(to + j * group * V), p);
          else
            st_part(to + j * group * V, p, part.at(j));
        } else if ((j * group + G.tid) * V < d) {
          st_once(reinterpret_cast<P*>(to + j * group * V), p);
        }
      }
      if (G.tid == 0) {
        if (mean) mean[(r + k) * mine.period] = s[k];
        if (rstd) rstd[(r + k) * mine.period] = rs;
      }
    }
  }
}

// The gradient: dx, and where work is given this block's sums of dy*h and dy
// as rows 2*block and 2*block + 1 of it (the groups add theirs in order).
template <typename T, typename TW, int V, int EACH, int ROWS, bool SUB, int EDGE>
__global__ void __launch_bounds__(kFlow, 1)
    norm_grad_flow_kernel(const MapalNormSite S, const T* x, const void* __restrict__ w, const float* __restrict__ mean,
                          const float* __restrict__ rstd, const T* dy, T* dx, float* __restrict__ work, int group,
                          uint32_t period) {
  using R = std::conditional_t<EDGE != 0, EdgeRing<T, EACH, ROWS, 2, SUB, EDGE == 2>, Ring<T, V, EACH, ROWS, 2>>;
  using P = Pack<T, V>;
  constexpr int NV = EACH / V, H = EACH / 2;
  __shared__ float sets[kMostGroups][2][2 * ROWS][16];
  extern __shared__ __align__(16) uint8_t dyn[];
  float* sums = reinterpret_cast<float*>(dyn);  // 2*d floats, when the ring is done
  const Group<SUB> G(group);
  R ring(dyn, G);
  auto* red = sets[SUB || group == 32 ? 0 : G.id];
  const Turns<SUB, EDGE, ROWS> mine(G, period, S.rows);
  uint64_t rows = mine.rows, ldx = mine.stride(S.ldx), lddy = mine.stride(S.lddy), lddx = mine.stride(S.lddx);
  uint64_t r = mine.first;
  const int d = (int)S.d, shift = mine.template shift<T>(S.lddx);
  const int shift_x = mine.template shift<T>(S.ldx), shift_y = mine.template shift<T>(S.lddy);
  using In = std::conditional_t<EDGE != 0, Input<V, NV>, Whole>;
  const In ix(group, G.tid, d, shift_x, shift), iy(group, G.tid, d, shift_y, shift);
  const std::conditional_t<EDGE != 0, Mine<V, NV>, Whole> part(group, G.tid, shift, d + shift);
  const std::conditional_t<EDGE != 0, Masks<P, V, NV>, Whole> keep(part);
  x = mine.at(x, S.ldx) - shift_x + (G.tid - ix.back) * V;
  dy = mine.at(dy, S.lddy) - shift_y + (G.tid - iy.back) * V;
  dx = mine.at(dx, S.lddx) - shift + G.tid * V;
  mean = mine.at(mean, 1);
  rstd = mine.at(rstd, 1);
  if constexpr (EDGE != 0) {
    pin(x), pin(dy), pin(dx);
    pin(rows), pin(ldx), pin(lddy), pin(lddx);
  }
  const float inv_n = __fdiv_rn(1.0f, (float)d);
  auto start = [&](int st, uint64_t row) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (row + k < rows) {
        const T* from = x + (row + k) * ldx;
        const T* from2 = dy + (row + k) * lddy;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if constexpr (EDGE != 0) {
            ring.bring(st, k * NV + j, from + j * group * V, ix.left[j]);
            ring.bring(st, (ROWS + k) * NV + j, from2 + j * group * V, iy.left[j]);
          } else if ((j * group + G.tid) * V < d) {
            ring.copy(st, k * NV + j, from + j * group * V);
            ring.copy(st, (ROWS + k) * NV + j, from2 + j * group * V);
          }
        }
      }
    ring.commit();
  };
  grid_wait();
  grid_go();
#pragma unroll
  for (int k = 0; k < R::kStages; ++k) start(k, r + k * mine.step);
  float nmu[ROWS], nrs[ROWS];
  auto stats = [&](uint64_t row) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const bool in = row + k < rows;
      nmu[k] = in ? __ldg(mean + (row + k) * mine.period) : 0.0f;
      nrs[k] = in ? __ldg(rstd + (row + k) * mine.period) : 0.0f;
    }
  };
  stats(r);
  f2 fw[H], aw[H], ab[H];
  {
    float a[EACH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * group + G.tid) * V;
      float pa[V] = {};
      if constexpr (EDGE != 0)
        weights_at<TW, V>(w, i - shift, d, 1.0f, pa);
      else if (i < d)
        weights<TW, V>(w, i, 1.0f, pa);
#pragma unroll
      for (int e = 0; e < V; ++e) a[j * V + e] = pa[e];
    }
#pragma unroll
    for (int u = 0; u < H; ++u) {
      fw[u] = f2_pack(a[2 * u], a[2 * u + 1]);
      aw[u] = ab[u] = f2_splat(0.0f);
    }
  }
  int par = 0;
  for (; r < rows; r += mine.step, par ^= 1) {
    ring.wait();
    f2 h[ROWS][H], g[ROWS][H];
    float c[2 * ROWS], rs[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      float fx[EACH], fy[EACH];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        P px, py;
        if constexpr (EDGE != 0) {
          px = ring.take(k * NV + j, ix.by);
          py = ring.take((ROWS + k) * NV + j, iy.by);
          keep(px, j);
          keep(py, j);
          if (r + k >= rows) {  // they are added to the sums over rows
            px.clear();
            py.clear();
          }
        } else if ((j * group + G.tid) * V < d && r + k < rows) {
          px = ring.take(k * NV + j);
          py = ring.take((ROWS + k) * NV + j);
        } else {
          px.clear();
          py.clear();
        }
        float a[V], e2[V];
        px.get(a);
        py.get(e2);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          fx[j * V + e] = a[e];
          fy[j * V + e] = e2[e];
        }
      }
      rs[k] = nrs[k];
      const f2 m = f2_splat(-nmu[k]), sc = f2_splat(nrs[k]);
      f2 c1 = f2_splat(0.0f), c2 = c1;
#pragma unroll
      for (int u = 0; u < H; ++u) {
        const f2 t = f2_pack(fy[2 * u], fy[2 * u + 1]);
        h[k][u] = f2_mul(f2_add(f2_pack(fx[2 * u], fx[2 * u + 1]), m), sc);
        g[k][u] = f2_mul(t, fw[u]);
        aw[u] = f2_fma(t, h[k][u], aw[u]);
        ab[u] = f2_add(ab[u], t);
        c1 = f2_add(c1, g[k][u]);
        c2 = f2_fma(g[k][u], h[k][u], c2);
      }
      c[2 * k] = f2_sum(c1);
      c[2 * k + 1] = f2_sum(c2);
    }
    stats(r + mine.step);
    G.sums(c, red[par]);
    if constexpr (EDGE != 0) ring.taken();
    start(ring.stage, r + R::kStages * mine.step);  // this turn's slots have been read
    ring.next_stage();
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (r + k >= rows) break;
      const f2 c1 = f2_splat(-c[2 * k] * inv_n), c2 = f2_splat(-c[2 * k + 1] * inv_n), sc = f2_splat(rs[k]);
      float f[EACH];
#pragma unroll
      for (int u = 0; u < H; ++u) {
        const f2 o = f2_mul(f2_fma(h[k][u], c2, f2_add(g[k][u], c1)), sc);
        f[2 * u] = f2_lo(o);
        f[2 * u + 1] = f2_hi(o);
      }
      T* to = dx + (r + k) * lddx;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = f[j * V + e];
        P p;
        p.set(o);
        if constexpr (EDGE != 0) {
          if (part.at(j) == part.kAll)
            st_once(reinterpret_cast<P*>(to + j * group * V), p);
          else
            st_part(to + j * group * V, p, part.at(j));
        } else if ((j * group + G.tid) * V < d) {
          st_once(reinterpret_cast<P*>(to + j * group * V), p);
        }
      }
    }
  }
  if (!work) return;
  // groups of one warp first, then warps or larger groups in order
  if constexpr (SUB) {
    __syncwarp();
    for (int o = group; o < 32; o <<= 1)
#pragma unroll
      for (int u = 0; u < H; ++u) {
        aw[u] = f2_add(aw[u], __shfl_xor_sync(0xffffffffu, aw[u], o));
        ab[u] = f2_add(ab[u], __shfl_xor_sync(0xffffffffu, ab[u], o));
      }
  }
  const int turns = blockDim.x / (SUB ? 32 : group);
  const int turn = !SUB ? G.id : (int)(threadIdx.x % 32) < group ? (int)(threadIdx.x / 32) : -1;
  float* out = work + 2ull * blockIdx.x * S.d;
  __syncthreads();  // every group has taken its last rows out of the ring
  for (int k = 0; k < turns; ++k) {
    if (turn == k) {
      const bool first = k == 0, last = k == turns - 1;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (j * group + G.tid) * V - shift;
        if (i >= d) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if constexpr (EDGE != 0)
            if (!(part.at(j) & (1u << e))) continue;
          const int u = j * V + e;
          const float a = u % 2 ? f2_hi(aw[u / 2]) : f2_lo(aw[u / 2]), c = u % 2 ? f2_hi(ab[u / 2]) : f2_lo(ab[u / 2]);
          (last ? out : sums)[i + e] = first ? a : sums[i + e] + a;
          (last ? out : sums)[d + i + e] = first ? c : sums[d + i + e] + c;
        }
      }
    }
    __syncthreads();
  }
}

// ---- longer rows -------------------------------------------------------------------
//
// One block a row, which is read again for each pass (from L1 or L2: rows of a
// few hundred KB); sums over rows by column, with partial sums in `work`.

template <typename T, typename TW, int V>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(const MapalNormSite S, const T* x, const void* w,
                                                             const void* b, T* y, float* mean, float* rstd) {
  __shared__ float red[2][32];
  const int64_t d = (int64_t)S.d;
  const float n = (float)S.d;
  grid_wait();
  grid_go();
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x) {
    const T* xr = x + r * S.ldx;
    T* yr = y + r * S.ldy;
    float s = 0.0f;
    for (int64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
      float f[V];
      reinterpret_cast<const Pack<T, V>*>(xr + i)->get(f);
#pragma unroll
      for (int e = 0; e < V; ++e) s += f[e];
    }
    const float mu = __fdiv_rn(block_sum(s, red[0]), n);
    float q = 0.0f;
    for (int64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
      float f[V];
      reinterpret_cast<const Pack<T, V>*>(xr + i)->get(f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float c = f[e] - mu;
        q = __fmaf_rn(c, c, q);
      }
    }
    const float rs = inv_std(__fdiv_rn(block_sum(q, red[1]), n), S.eps);
    for (int64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
      float f[V], fw[V], fb[V];
      reinterpret_cast<const Pack<T, V>*>(xr + i)->get(f);
      weights<TW, V>(w, i, 1.0f, fw);
      weights<TW, V>(b, i, 0.0f, fb);
      Pack<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = __fmaf_rn((f[e] - mu) * rs, fw[e], fb[e]);
      o.set(f);
      st_once(reinterpret_cast<Pack<T, V>*>(yr + i), o);
    }
    if (threadIdx.x == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <typename T, typename TW, int V>
__global__ void __launch_bounds__(kThreads) norm_grad_rows_kernel(const MapalNormSite S, const T* x, const void* w,
                                                                  const float* mean, const float* rstd, const T* dy,
                                                                  T* dx) {
  __shared__ float red[2][2][32];
  const int64_t d = (int64_t)S.d;
  const float n = (float)S.d;
  grid_wait();
  grid_go();
  int par = 0;
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x, par ^= 1) {
    const T* xr = x + r * S.ldx;
    const T* dyr = dy + r * S.lddy;
    const float mu = mean[r], rs = rstd[r];
    float c1 = 0.0f, c2 = 0.0f;
    for (int64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
      float fx[V], fy[V], fw[V];
      reinterpret_cast<const Pack<T, V>*>(xr + i)->get(fx);
      reinterpret_cast<const Pack<T, V>*>(dyr + i)->get(fy);
      weights<TW, V>(w, i, 1.0f, fw);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = fy[e] * fw[e];
        c1 += g;
        c2 = __fmaf_rn(g, (fx[e] - mu) * rs, c2);
      }
    }
    c1 = __fdiv_rn(block_sum(c1, red[par][0]), n);
    c2 = __fdiv_rn(block_sum(c2, red[par][1]), n);
    for (int64_t i = threadIdx.x * V; i < d; i += kThreads * V) {
      float fx[V], fy[V], fw[V];
      reinterpret_cast<const Pack<T, V>*>(xr + i)->get(fx);
      reinterpret_cast<const Pack<T, V>*>(dyr + i)->get(fy);
      weights<TW, V>(w, i, 1.0f, fw);
      Pack<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) fx[e] = __fmaf_rn(-((fx[e] - mu) * rs), c2, fy[e] * fw[e] - c1) * rs;
      o.set(fx);
      st_once(reinterpret_cast<Pack<T, V>*>(dx + r * S.lddx + i), o);
    }
  }
}

// dx of rows that a block's registers hold as they were read, EACH elements of
// x and of dy a thread, with the weights in shared memory (f32 weights of 16384
// columns do not stay in L1 beside the rows: 300 us for 8000 rows of bf16). Two
// blocks an SM hide each other's barriers. 8000 x 16384 bf16 156 us, the kernel
// above 396.
template <typename T, typename TW, int V, int EACH>
__global__ void __launch_bounds__(1024) norm_grad_held_kernel(const MapalNormSite S, const T* x, const TW* w,
                                                              const float* mean, const float* rstd, const T* dy, T* dx) {
  using P = Pack<T, V>;
  constexpr int NV = EACH / V;
  __shared__ float red[2][2][32];
  extern __shared__ __align__(16) uint8_t dyn[];  // d weights
  const int d = (int)S.d, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float n = (float)d;
  int par = 0;
  grid_wait();
  grid_go();
  if (w) {
    using U = Pack<TW, (V * sizeof(TW) > 16 ? 16 / sizeof(TW) : V)>;
    constexpr int kU = sizeof(U) / sizeof(TW);
#pragma unroll 4
    for (int i = threadIdx.x; i < d / kU; i += blockDim.x) reinterpret_cast<U*>(dyn)[i] = reinterpret_cast<const U*>(w)[i];
    w = reinterpret_cast<const TW*>(dyn);
    __syncthreads();
  }
  for (uint64_t r = blockIdx.x; r < S.rows; r += gridDim.x, par ^= 1) {
    P a[NV], b[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * blockDim.x + threadIdx.x) * V;
      if (i < d) {
        a[j] = ld_once(reinterpret_cast<const P*>(x + r * S.ldx + i));
        b[j] = ld_once(reinterpret_cast<const P*>(dy + r * S.lddy + i));
      } else {
        a[j].clear();
        b[j].clear();
      }
    }
    const float mu = __ldg(mean + r), rs = __ldg(rstd + r);
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * blockDim.x + threadIdx.x) * V;
      if (i < d) {
        float fx[V], fy[V], fw[V];
        a[j].get(fx);
        b[j].get(fy);
        weights<TW, V>(w, i, 1.0f, fw);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float g = fy[e] * fw[e];
          c1 += g;
          c2 = __fmaf_rn(g, (fx[e] - mu) * rs, c2);
        }
      }
      asm volatile("" ::: "memory");  // keeps the weights' loads from piling up in registers
    }
    c1 = warp_sum(c1);
    c2 = warp_sum(c2);
    if (lane == 0) {
      red[par][0][warp] = c1;
      red[par][1][warp] = c2;
    }
    __syncthreads();
    c1 = __fdiv_rn(warp_sum(lane < warps ? red[par][0][lane] : 0.0f), n);
    c2 = __fdiv_rn(warp_sum(lane < warps ? red[par][1][lane] : 0.0f), n);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * blockDim.x + threadIdx.x) * V;
      if (i < d) {
        a[j].forget();
        b[j].forget();
        float fx[V], fy[V], fw[V];
        a[j].get(fx);
        b[j].get(fy);
        weights<TW, V>(w, i, 1.0f, fw);
        P o;
#pragma unroll
        for (int e = 0; e < V; ++e) fx[e] = __fmaf_rn(-((fx[e] - mu) * rs), c2, fy[e] * fw[e] - c1) * rs;
        o.set(fx);
        st_once(reinterpret_cast<P*>(dx + r * S.lddx + i), o);
      }
      asm volatile("" ::: "memory");
    }
  }
}

// dw and db over rows p*8 + sub, then every parts*8-th: part p's sums of 32*V
// columns. A row is a whole number of packs (V divides d).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_grad_cols_kernel(const MapalNormSite S, const T* x, const float* mean,
                                                                  const float* rstd, const T* dy, float* work,
                                                                  uint32_t parts) {
  __shared__ float sw[8][32 * V], sb[8][32 * V];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint64_t c = ((uint64_t)blockIdx.x * 32 + lane) * V;
  float aw[V] = {}, ab[V] = {};
  grid_wait();
  grid_go();
  if (c < S.d)
    for (uint64_t r = blockIdx.y * 8ull + sub; r < S.rows; r += parts * 8ull) {
      const Pack<T, V> p = ld_once(reinterpret_cast<const Pack<T, V>*>(x + r * S.ldx + c));
      const Pack<T, V> t = ld_once(reinterpret_cast<const Pack<T, V>*>(dy + r * S.lddy + c));
      const float mu = __ldg(mean + r), rs = __ldg(rstd + r);
      float fx[V], fy[V];
      p.get(fx);
      t.get(fy);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = fy[e];
        aw[e] = __fmaf_rn(g, (fx[e] - mu) * rs, aw[e]);
        ab[e] += g;
      }
    }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sw[sub][e * 32 + lane] = aw[e];
    sb[sub][e * 32 + lane] = ab[e];
  }
  __syncthreads();
  if (sub == 0 && c < S.d) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      for (int k = 1; k < 8; ++k) {
        aw[e] += sw[k][e * 32 + lane];
        ab[e] += sb[k][e * 32 + lane];
      }
      work[(2ull * blockIdx.y) * S.d + c + e] = aw[e];
      work[(2ull * blockIdx.y + 1) * S.d + c + e] = ab[e];
    }
  }
}

// dw and db from the parts' sums: 32 runs of parts in order, then the runs. No parts: zeros.
__global__ void __launch_bounds__(1024) norm_grad_join_kernel(const float* __restrict__ work, uint64_t d,
                                                                  uint32_t parts, float* dw, float* db) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;  // 0..d: dw, d..2d: db
  float a = 0.0f;
  grid_wait();
  grid_go();
  if (c < 2 * d) {
#pragma unroll 10
    for (uint32_t p = sub; p < parts; p += 32) a += __ldcs(work + 2ull * p * d + c);
  }
  red[lane][sub] = a;
  __syncthreads();
  a = warp_sum(red[sub][lane]);  // warp `sub` joins column `sub`
  const uint64_t o = (uint64_t)blockIdx.x * 32 + sub;
  if (lane == 0 && o < 2 * d) {
    float* out = o < d ? dw : db;
    if (out) out[o < d ? o : o - d] = a;
  }
}

// ---- host --------------------------------------------------------------------------

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

// Partial sums that the gradient's scratch has room for: a block each (up to 7
// more than rows, so that their number suits every period), and for longer rows
// as many as give 16 blocks an SM or more.
uint32_t grad_parts(const MapalNormSite& s, int sms) {
  const uint64_t want = s.d <= kMostFlow ? s.rows + 7 : (s.rows + 7) / 8,
                 cap = s.d <= kMostFlow ? sms : (16ull * sms * 256 + s.d - 1) / s.d;
  return (uint32_t)(want < 1 ? 1 : want < cap ? want : cap);
}

uint64_t grad_bytes(const MapalNormSite& s, int sms) { return grad_parts(s, sms) * 2ull * s.d * sizeof(float); }

unsigned row_blocks(const MapalNormSite& s, int sms) { return (unsigned)(s.rows < 8ull * sms ? s.rows : 8ull * sms); }

template <typename T, typename TW, int V, int EACH>
int launch_held(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const void* b, void* y,
                 float* mean, float* rstd) {
  const int group = (int)((s.d + 32 * EACH - 1) / (32 * EACH)) * 32;
  // one row a block while that leaves no SM with two
  const int threads = group >= 256 || s.rows <= (uint64_t)D.prof.sm_count ? group : 256 / group * group;
  const uint64_t want = (s.rows + threads / group - 1) / (threads / group),
                 cap = (uint64_t)D.prof.sm_count * (1024 / threads);
  return launch_rows(norm_held_kernel<T, TW, V, EACH>, (unsigned)(want < cap ? want : cap), threads, 0, D.stream, 1, s,
                     (const T*)x, w, b, (T*)y, mean, rstd, group);
}

template <typename T, typename TW, int V, int EACH, int ROWS, bool SUB, int EDGE = 0>
int launch_flow(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const void* b, void* y,
                float* mean, float* rstd) {
  constexpr size_t smem =
      std::conditional_t<EDGE != 0, EdgeRing<T, EACH, ROWS, 1, SUB, EDGE == 2>, Ring<T, V, EACH, ROWS, 1>>::kBytes;
  static std::atomic<uint64_t> done{0};
  auto kernel = norm_flow_kernel<T, TW, V, EACH, ROWS, SUB, EDGE>;
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, smem, "layer_norm shared memory"));
  const uint32_t period = EDGE ? edge_period(s.rows, {s.ldx, s.ldy}, V) : 1;
  const Plan p = flow_plan(s.rows, EDGE ? s.d + V - 1 : s.d, D.prof.sm_count, EACH, ROWS, period);
  return launch_rows(kernel, p.blocks, p.threads, smem, D.stream, 1, s, (const T*)x, w, b, (T*)y, mean, rstd, p.group,
                     period);
}

template <typename T, typename TW, int V, int EDGE>
int launch_norm(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const void* b, void* y,
                float* mean, float* rstd) {
  constexpr int kMid = V == 1 ? 16 : 32;
  constexpr int kLong = V == 1 ? 16 : 32;
  // Many rows: a thread of the device gets at least two turns of 32 elements
  // (eight where it loads them one by one and a turn is slower to start).
  const bool many = s.rows * s.d >= (V == 1 ? 256ull : 64ull) * kFlow * D.prof.sm_count;
  // 16-byte accesses of 16-bit types do better with 16 columns a thread (and
  // half the warps at each barrier) from 512 columns on: 16384 x 4096 bf16 52
  // against 60 us, 60000 x 1024 45 against 54; f32 and narrow accesses do not.
  constexpr uint64_t kNarrow = sizeof(T) * V == 16 && sizeof(T) == 2 ? 512 : 4096;
  if constexpr (EDGE != 0) {
    const uint64_t span = s.d + V - 1;
    if (span <= 128) return launch_flow<T, TW, V, 8, 4, true, EDGE>(D, s, x, w, b, y, mean, rstd);
    if (span > kMostFlow) return launch_flow<T, TW, V, 32, 1, false, EDGE>(D, s, x, w, b, y, mean, rstd);
    // whichever has more rows at once, which is what a span just over a whole
    // number of warps decides (60000 x 1021: 93 us, with 16 columns a thread 100)
    const uint64_t wide = rows_at_once(span, 16, 2), narrow = span <= 4096 ? rows_at_once(span, 8, 4) : 0;
    if (span <= kNarrow ? narrow >= wide : narrow > wide)
      return launch_flow<T, TW, V, 8, 4, false, EDGE>(D, s, x, w, b, y, mean, rstd);
    return launch_flow<T, TW, V, 16, 2, false, EDGE>(D, s, x, w, b, y, mean, rstd);
  } else if (s.d <= 128 && many)
    return launch_flow<T, TW, V, 8, 4, true>(D, s, x, w, b, y, mean, rstd);
  else if (s.d <= kNarrow && many)
    return launch_flow<T, TW, V, 8, 4, false>(D, s, x, w, b, y, mean, rstd);
  else if (s.d <= kMostFlow && many)
    return launch_flow<T, TW, V, 16, 2, false>(D, s, x, w, b, y, mean, rstd);
  else if (V > 1 && s.d <= 2 * kMostFlow && many)
    return launch_flow<T, TW, V, kLong, 32 / kLong, false>(D, s, x, w, b, y, mean, rstd);
  else if (s.d <= 1024 * 8)
    return launch_held<T, TW, V, 8>(D, s, x, w, b, y, mean, rstd);
  else if (s.d <= 1024 * kMid)
    return launch_held<T, TW, V, kMid>(D, s, x, w, b, y, mean, rstd);
  else
    return launch_rows(norm_rows_kernel<T, TW, V>, row_blocks(s, D.prof.sm_count), kThreads, 0, D.stream, 1, s,
                       (const T*)x, w, b, (T*)y, mean, rstd);
}

template <typename T, typename TW, int V, int EACH, int ROWS, bool SUB, int EDGE>
int launch_grad_flow(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const float* mean,
                     const float* rstd, const void* dy, void* dx, float* work, uint32_t& parts) {
  constexpr size_t ring =
      std::conditional_t<EDGE != 0, EdgeRing<T, EACH, ROWS, 2, SUB, EDGE == 2>, Ring<T, V, EACH, ROWS, 2>>::kBytes;
  static std::atomic<uint64_t> done{0};
  auto kernel = norm_grad_flow_kernel<T, TW, V, EACH, ROWS, SUB, EDGE>;
  const uint32_t period = EDGE ? edge_period(s.rows, {s.ldx, s.lddy, s.lddx}, V) : 1;
  const Plan p = flow_plan(s.rows, EDGE ? s.d + V - 1 : s.d, D.prof.sm_count, EACH, ROWS, period);
  parts = p.blocks;
  const size_t sums = p.threads > p.group ? 2 * s.d * sizeof(float) : 0;  // at most 32 KB: d <= 4096
  MAPAL_TRY(ensure_smem_attr(done, (const void*)kernel, D.device, ring > 32768 ? ring : 32768,
                             "layer_norm_grad shared memory"));
  return launch_rows(kernel, p.blocks, p.threads, ring > sums ? ring : sums, D.stream, 1, s, (const T*)x, w, mean, rstd,
                     (const T*)dy, (T*)dx, work, p.group, period);
}

template <typename T, typename TW, int V, int EDGE>
int launch_norm_grad(const DeviceSlot& D, const MapalNormSite& s, const void* x, const void* w, const float* mean,
                     const float* rstd, const void* dy, void* dx, float* dw, float* db, float* work) {
  const int sms = D.prof.sm_count;
  uint32_t parts = grad_parts(s, sms);
  if (!dw && !db) work = nullptr;
  const bool flow = s.d <= kMostFlow && s.rows;
  // as in the forward pass, but more registers hang on a column: 16384 x 4096
  // bf16 75 against 77 us, 60000 x 1024 73 against 69
  constexpr uint64_t kNarrow = sizeof(T) * V == 16 && sizeof(T) == 2 ? 2048 : 4096;
  const uint64_t span = EDGE ? s.d + V - 1 : s.d;
  if (flow && span <= 128) {
    MAPAL_TRY((launch_grad_flow<T, TW, V, 8, 2, true, EDGE>(D, s, x, w, mean, rstd, dy, dx, work, parts)));
  } else if (flow && (EDGE ? span <= 4096 && rows_at_once(span, 8, 2) >= rows_at_once(span, 16, 1) : span <= kNarrow)) {
    MAPAL_TRY((launch_grad_flow<T, TW, V, 8, 2, false, EDGE>(D, s, x, w, mean, rstd, dy, dx, work, parts)));
  } else if (flow) {
    MAPAL_TRY((launch_grad_flow<T, TW, V, 16, 1, false, EDGE>(D, s, x, w, mean, rstd, dy, dx, work, parts)));
  } else if (s.rows == 0) {
    parts = 0;  // sums over no rows: the join writes zeros and reads nothing
  } else if constexpr (EDGE == 0) {
    // rows of more than kMostFlow elements, which are whole accesses (V divides d): edge_rows takes none of them
    if (work)  // before dx is written, which may be dy
      MAPAL_TRY(launch_rows(norm_grad_cols_kernel<T, V>, dim3((unsigned)((s.d + 32 * V - 1) / (32 * V)), parts), kThreads,
                            0, D.stream, 1, s, (const T*)x, mean, rstd, (const T*)dy, work, parts));
  }
  if (work)
    MAPAL_TRY(launch_rows(norm_grad_join_kernel, (unsigned)((2 * s.d + 31) / 32), 1024, 0, D.stream, 1, work, s.d, parts, dw,
                          db));
  if constexpr (EDGE == 0) {
    constexpr int kHeld = sizeof(T) * V == 16 && sizeof(T) == 2 ? 32 : 16;
    if (!flow && s.rows && s.d <= 1024 * kHeld) {
      const int threads = (int)((s.d + 32 * kHeld - 1) / (32 * kHeld)) * 32;
      static std::atomic<uint64_t> done{0};
      MAPAL_TRY(ensure_smem_attr(done, (const void*)norm_grad_held_kernel<T, TW, V, kHeld>, D.device,
                                 1024 * kHeld * sizeof(TW), "layer_norm_grad shared memory"));
      const uint64_t cap = (uint64_t)sms * (1024 / threads);
      MAPAL_TRY(launch_rows(norm_grad_held_kernel<T, TW, V, kHeld>, (unsigned)(s.rows < cap ? s.rows : cap), threads,
                            w ? s.d * sizeof(TW) : 0, D.stream, 1, s, (const T*)x, (const TW*)w, mean, rstd, (const T*)dy,
                            (T*)dx));
    } else if (!flow && s.rows) {
      MAPAL_TRY(launch_rows(norm_grad_rows_kernel<T, TW, V>, row_blocks(s, sms), kThreads, 0, D.stream, 1, s, (const T*)x,
                            w, mean, rstd, (const T*)dy, (T*)dx));
    }
  }
  return 0;
}

// f(T, TW, V, EDGE) for the site's types and the widest access (16, 4 or an
// element's bytes) that a row is a multiple of and all arrays' rows begin at;
// edge (1 or 2): 16 bytes whatever the rows are, instead of single elements.
// Pairs of 16-bit elements do without (30000 x 2046 bf16 74 and 101 us, with it
// 75 and 137).
template <typename F>
int by_type(const MapalNormSite& s, int width, int edge, const void* w, const void* b, F&& f0) {
  using std::integral_constant;
  const int ww = align_of(w, 0, 1) < align_of(b, 0, 1) ? align_of(w, 0, 1) : align_of(b, 0, 1);
  const int ws = dtype_bytes(s.wtype);
  if (width >= (s.dtype == MAPAL_DTYPE_F32 ? 16 : 4) || ww < 16) edge = 0;
  auto f = [&](auto t, auto tw, auto v) {
    if constexpr (v.value * sizeof(t) == 16) {
      if (edge == 1) return f0(t, tw, v, integral_constant<int, 1>{});
      if (edge == 2) return f0(t, tw, v, integral_constant<int, 2>{});
    }
    return f0(t, tw, v, integral_constant<int, 0>{});
  };
  if (edge) width = 16;
  if (s.dtype == MAPAL_DTYPE_F32) {
    if (width >= 16 && ww >= 16) return f(float{}, float{}, integral_constant<int, 4>{});
    return f(float{}, float{}, integral_constant<int, 1>{});
  }
  auto half = [&](auto t, auto tw) {
    if (width >= 16 && ww >= 16) return f(t, tw, integral_constant<int, 8>{});
    if (width >= 4 && ww >= 2 * ws) return f(t, tw, integral_constant<int, 2>{});
    return f(t, tw, integral_constant<int, 1>{});
  };
  const bool wide = s.wtype == MAPAL_DTYPE_F32;
  if (s.dtype == MAPAL_DTYPE_F16) return wide ? half(__half{}, float{}) : half(__half{}, __half{});
  return wide ? half(__nv_bfloat16{}, float{}) : half(__nv_bfloat16{}, __nv_bfloat16{});
}

// Whether the kernels for rows at odd places take these (arrays that begin at
// a 16-byte boundary, rows that fit), and which: 1 where the inputs' rows begin
// as the output's do, 2 where they are shifted.
template <typename... A>
int edge_rows(const MapalNormSite& s, uint64_t most, std::initializer_list<uint64_t> ins, uint64_t out, A... arrays) {
  const uint64_t v = 16 / dtype_bytes(s.dtype);
  if (s.d + v - 1 > most || !(aligned16(arrays) && ...)) return 0;
  for (const uint64_t ld : ins)
    if (s.rows > 1 && (ld - out) % v != 0) return 2;
  return 1;
}

int narrowest(std::initializer_list<int> widths) {
  int w = 16;
  for (const int o : widths) w = o < w ? o : w;
  return w;
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
    if (x == y && site->rows > 1 && site->ldx != site->ldy)
      return set_error(MAPAL_ERR_INVALID, "y is x, but not at the same stride");
    if (!aligned_to(x, es) || !aligned_to(y, es) || !aligned_to(w, ws) || !aligned_to(b, ws) ||
        !aligned_to(mean, 4) || !aligned_to(rstd, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    const int width = narrowest({align_of(x, site->ldx * es, site->rows), align_of(y, site->ldy * es, site->rows),
                                 align_of(nullptr, site->d * es, 2)});
    const DeviceSlot& D = ctx->dev[0];
    const bool few = site->rows * site->d < kEdgeTurns * kFlow * D.prof.sm_count;
    const int edge = few ? 0 : edge_rows(*site, 2 * kMostFlow, {site->ldx}, site->ldy, x, y);
    MAPAL_TRY(by_type(*site, width, edge, w, b, [&](auto t, auto tw, auto v, auto e) {
      return launch_norm<decltype(t), decltype(tw), v.value, e.value>(D, *site, x, w, b, y, mean, rstd);
    }));
    return finish(ctx, 0, false);
  });
}

extern "C" int mapal_gpu_layer_norm_grad_workspace(MapalGpuCtx* ctx, const MapalNormSite* site, uint64_t* bytes) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_norm(site));
    if (!bytes) return set_error(MAPAL_ERR_INVALID, "bytes is null");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
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
    if (site->rows > 1 && ((dx == dy && site->lddx != site->lddy) || (dx == x && site->lddx != site->ldx)))
      return set_error(MAPAL_ERR_INVALID, "dx is dy or x, but not at the same stride");
    if (!aligned_to(x, es) || !aligned_to(dy, es) || !aligned_to(dx, es) || !aligned_to(w, ws) ||
        !aligned_to(mean, 4) || !aligned_to(rstd, 4) || !aligned_to(dw, 4) || !aligned_to(db, 4))
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    if ((dw || db) && (!work || !aligned16(work)))
      return set_error(MAPAL_ERR_INVALID, "work is null or not 16-byte aligned");
    if (site->rows == 0 && !dw && !db) return 0;
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    if ((dw || db) && work_bytes < grad_bytes(*site, ctx->dev[0].prof.sm_count))
      return set_error(MAPAL_ERR_INVALID, "work is shorter than mapal_gpu_layer_norm_grad_workspace says");
    const int width = narrowest({align_of(x, site->ldx * es, site->rows), align_of(dy, site->lddy * es, site->rows),
                                 align_of(dx, site->lddx * es, site->rows), align_of(nullptr, site->d * es, 2)});
    // a few longer rows have more threads one by one (300 x 4091 bf16 11.4 us, 13.8)
    const DeviceSlot& D = ctx->dev[0];
    const bool few = site->d > 2040 && site->rows * site->d < 64ull * kFlow * D.prof.sm_count;
    const int edge = few ? 0 : edge_rows(*site, kMostFlow, {site->ldx, site->lddy}, site->lddx, x, dy, dx);
    MAPAL_TRY(by_type(*site, width, edge, w, w, [&](auto t, auto tw, auto v, auto e) {
      return launch_norm_grad<decltype(t), decltype(tw), v.value, e.value>(D, *site, x, w, mean, rstd, dy, dx, dw,
                                                                            db, (float*)work);
    }));
    return finish(ctx, 0, false);
  });
}

// linear_loss.cu — the softmax cross entropy of a vocabulary's logits, from the rows
// before them and the vocabulary's weights (mapal_gpu_linear_loss*). No counterpart
// in the reference.
//
// With l_iv = <h_i, w_v>, m_i = max over v != t_i and s_i = sum over v != t_i of
// exp(l_iv - m_i), and u_i = max(m_i, l_it):
//   loss_i = (u_i - l_it) + log1p(s_i exp(m_i - u_i) + (exp(l_it - u_i) - 1))
//   lse_i  = u_i + the same log1p
// Both terms are never negative, and where the target is nearly certain (u = l_it)
// the argument is the others' sum alone: nothing cancels. The target's logit is a
// dot product of its own in f32. The gradient
//   dl_iv = g_i (exp(l_iv - lse_i) - [v = t_i]),  dh_i = sum_v dl_iv w_v,  dw_v = sum_i dl_iv h_i
// takes the logits again, a piece of the vocabulary at a time, as one 16-bit matrix
// dl from which both sums are products. The logits are never in memory.
// The target's own p - 1 is expm1(l_it - lse_i) with the logit that lse was made of, the
// same dot product: where the target is nearly certain, another sum of the same
// products is off by more than p - 1 is.
//
// Bound by the tensor cores: 2 rows*vocab*d operations forward, three times that
// backward. The rows that a call takes come first of all, side by side (list, h):
// those with a target, and all of them where lse is asked for, which every row has.
// The others cost nothing and whatever they hold is not read.
// Measured on a B200, graph replays, forward and backward: 8192 rows, 128000 x 4096 bf16
// 6.6 and 20.6 ms (1.27 PFLOP/s over four products, at the power limit); 2401 rows,
// 50257 x 1000 222 and 643 us in bf16, 287 and 700 in f16; 3001 rows of which 600 have no
// target, f16, 331 (270 without lse) and 779 us; 16 rows, 50257 x 2048 bf16 58 and 161 us
// (the weights, once and three times: 32 and 96).
#include <algorithm>

#include "product.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- rows taken ------------------------------------------------------------------------
//
// The rows that have a target (all: every row), in order: list[c] = row, and their
// h, target (-1: none), log-sum and gradient side by side. count = {0, how many}, the
// offsets of one group. Each block counts the targets before its rows itself (they
// are few bytes), so no scan goes before. Rows that are not taken get what they are
// due: a loss of 0, or a gradient of zeros.

struct Taken {
  int32_t* list;
  int32_t* count;
  int32_t* target;
  float* lse;
  float* g;
  float* missing;  // the target's probability less 1
  unsigned* most;  // the bits of the largest |g| (f16 alone; 0 before)
  uint16_t* h;     // stride ld, zeros from d up to it
  uint64_t ld;
};
struct TakeArgs {
  const uint16_t* h;
  const void* w;  // backward
  const int32_t* targets;
  const float* lse;
  const float* dloss;
  float* loss_out;  // forward
  uint16_t* dh;     // backward, may be null
  uint64_t ldh, ldw, lddh, rows, d;
  uint32_t vocab, chunk;  // rows a block takes
  uint32_t grad, all, aligned;
  uint32_t wide;  // h's rows side by side and the weights can be read eight at a time
  unsigned* trap;
};

constexpr int kTakeThreads = 256;

__device__ __forceinline__ bool is_target(int32_t t, uint32_t vocab) { return (uint32_t)t < vocab; }

// A lane's share of a row's target logit, V elements an access. The loss and its gradient
// take the same V, so that both have the same bits.
template <typename T, int V>
__device__ __forceinline__ float target_dot(const T* h, const T* w, uint32_t d) {
  float dot = 0.0f;
#pragma unroll 4
  for (uint32_t e = (threadIdx.x & 31) * V; e < d; e += 32 * V) {
    float x[V], y[V];
    reinterpret_cast<const Pack<T, V>*>(h + e)->get(x);
    reinterpret_cast<const Pack<T, V>*>(w + e)->get(y);
#pragma unroll
    for (int k = 0; k < V; ++k) dot = __fmaf_rn(x[k], y[k], dot);
  }
  return dot;
}

template <typename E>
__global__ void __launch_bounds__(kTakeThreads) take_rows_kernel(const TakeArgs A, const Taken T) {
  __shared__ uint32_t sums[kTakeThreads / 32];
  __shared__ uint32_t total;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_wait();
  grid_go();
  const uint64_t lo = (uint64_t)blockIdx.x * A.chunk, hi = min(lo + A.chunk, A.rows);
  uint32_t n = 0;
  if (A.all)
    n = threadIdx.x == 0 ? (uint32_t)lo : 0;
  else
    for (uint64_t i = threadIdx.x; i < lo; i += kTakeThreads) n += is_target(__ldg(A.targets + i), A.vocab);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) sums[warp] = n;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t w = 0; w < kTakeThreads / 32; ++w) before += sums[w];
  // a warp a row; every warp walks all of the block's targets, 32 at a time
  uint32_t most = 0;
  for (uint64_t i0 = lo; i0 < hi; i0 += 32) {
    const uint64_t i = i0 + lane;
    const int32_t t = i < hi ? __ldg(A.targets + i) : -1;
    const bool ok = is_target(t, A.vocab);
    if (warp == 0 && !ok && t != -1) atomicMax(A.trap, kTrapOob);
    const uint32_t which = __ballot_sync(0xffffffffu, ok || (A.all && i < hi));
    const uint32_t c = before + __popc(which & ((1u << lane) - 1));
    before += __popc(which);
    if (warp == 0 && i < hi) {
      if (ok || A.all) {
        T.list[c] = (int32_t)i;
        T.target[c] = ok ? t : -1;
        if (A.grad) {
          const float g = A.dloss ? __ldg(A.dloss + i) : 1.0f;
          T.lse[c] = __ldg(A.lse + i);
          T.g[c] = g;
          most = max(most, __float_as_uint(fabsf(g)));
        }
      } else if (!A.grad) {
        A.loss_out[i] = 0.0f;
      }
    }
    for (uint32_t r = warp; r < 32 && i0 + r < hi; r += kTakeThreads / 32) {
      const bool take = (which >> r) & 1;
      const uint32_t to = __shfl_sync(0xffffffffu, c, r);
      const int32_t target = __shfl_sync(0xffffffffu, t, r);
      if (take) {
        const uint16_t* from = A.h + (i0 + r) * A.ldh;
        uint16_t* out = T.h + (uint64_t)to * T.ld;
        if (A.aligned) {  // ld is d rounded up to 8
#pragma unroll 4
          for (uint64_t e = lane * 8; e + 8 <= A.d; e += 256)
            *reinterpret_cast<uint4*>(out + e) = __ldcs(reinterpret_cast<const uint4*>(from + e));
          const uint64_t e = A.d / 8 * 8 + lane;
          if (e < T.ld) out[e] = e < A.d ? from[e] : (uint16_t)0;
        } else {
          for (uint64_t e = lane; e < T.ld; e += 32) out[e] = e < A.d ? __ldg(from + e) : (uint16_t)0;
        }
        if (A.grad) {
          __syncwarp();  // the row as it lies now, whatever its own place
          const E* h = reinterpret_cast<const E*>(out);
          const E* w = static_cast<const E*>(A.w) + (uint64_t)target * A.ldw;
          const float dot = warp_sum(A.wide ? target_dot<E, 8>(h, w, (uint32_t)A.d) : target_dot<E, 1>(h, w, (uint32_t)A.d));
          if (lane == 0) T.missing[to] = expm1f(dot - __ldg(A.lse + i0 + r));
        }
      } else if (A.dh) {
        uint16_t* out = A.dh + (i0 + r) * A.lddh;
        for (uint64_t e = lane; e < A.d; e += 32) out[e] = 0;
      }
    }
  }
  if (warp == 0) {
    if (T.most && A.grad) {
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0 && most) atomicMax(T.most, most);
    }
    if (lane == 0 && hi == A.rows) {  // the last block has counted them all
      T.count[0] = 0;
      T.count[1] = (int32_t)before;
    }
  }
}

// Weights at places that TMA cannot read: a piece of them at stride ld, a multiple of 8.
__global__ void __launch_bounds__(256) copy_weights_kernel(const uint16_t* __restrict__ w, uint64_t ldw, uint32_t rows,
                                                           uint32_t d, uint16_t* __restrict__ out, uint32_t ld) {
  grid_wait();
  grid_go();
  const uint32_t words = ld / 8;
  const uint64_t n = (uint64_t)rows * words;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i / words;
    const uint32_t c = (uint32_t)(i % words) * 8;
    const uint16_t* p = w + r * ldw + c;
    const uint32_t here = min(8u, d - c), sh = (uint32_t)(uintptr_t)p & 15;
    const uint4* q = reinterpret_cast<const uint4*>((uintptr_t)p - sh);  // the aligned words with one of the elements
    const uint4 v = straddle(__ldg(q), sh + 2 * here > 16 ? __ldg(q + 1) : make_uint4(0, 0, 0, 0), sh);
    uint32_t o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) o[k] = here >= 2 * k + 2 ? o[k] : here == 2 * k + 1 ? o[k] & 0xffffu : 0u;
    *reinterpret_cast<uint4*>(out + r * ld + c) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---- forward -------------------------------------------------------------------------

// The tensor cores cut a sum towards zero at each step of 16 products: in one sum over
// d = 4096 a logit loses 4e-6 of itself in the mean, and lse, which is an average of
// logits, the same. In runs of 256 elements (Out::kRun) whose sums are added in f32 the
// cut is of small sums.
constexpr int kLogitRun = 4;

// A tile of logits, rows on the lanes and 128 of the vocabulary's columns a warp:
// each thread keeps the running maximum of its row and the sum of exponentials
// against it, the target's column left out, and writes one pair. Against a maximum
// that is infinite the sum is of exp(l) itself: inf, or NaN with one among them.
struct SumTile {
  static constexpr int kRun = kLogitRun;
  float2* parts;  // [part][row]
  uint64_t ld;
  const int32_t* target;
  uint32_t v0, part0;

  __device__ __forceinline__ void put(const ProductArgs& P, const Job& j, float (&l)[kHalfTokens], uint32_t lane0,
                                      uint32_t from) const {
    const uint32_t lane = lane0 + (threadIdx.x & 31);
    const bool in = lane < P.lanes;
    const uint32_t end = min(from + kHalfTokens, j.cols);
    const int32_t mine = in ? __ldg(target + lane) - (int32_t)(v0 + j.col0) : -1;  // the target's column of this tile
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int q = 0; q < kHalfTokens / 32; ++q) {
      const uint32_t j0 = from + q * 32;
      if (j0 >= end) break;
      float f[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = l[q * 32 + i];
      if (j0 + 32 > end) {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = j0 + i < end ? f[i] : -INFINITY;
      }
      const uint32_t hit = (uint32_t)(mine - (int32_t)j0);
      if (any_of(hit < 32)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = hit == i ? -INFINITY : f[i];
      }
      float top = f[0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, f[i]);
      const float next = fmaxf(m, top);
      const float base = isinf(next) ? 0.0f : -next * kLog2e;
      float sum[4] = {};
#pragma unroll
      for (int i = 0; i < 32; ++i) sum[i & 3] += ex2(__fmaf_rn(f[i], kLog2e, base));
      s = __fmaf_rn(s, ex2(__fmaf_rn(m, kLog2e, base)), (sum[0] + sum[1]) + (sum[2] + sum[3]));
      m = next;
    }
    if (in) parts[(uint64_t)(part0 + j.col0 / 128 + from / 128) * ld + lane] = make_float2(m, s);
  }
};

// The parts of a row joined: 8 rows a block, 32 parts at a time, and a warp a row for its
// target's logit, whose loads run beside the others'.
constexpr int kJoinRows = 8, kJoinAhead = 4;

__device__ __forceinline__ void join(float2& a, const float2& b) {
  const float m = fmaxf(a.x, b.x);
  // -inf: no number on either side, sums of nothing, or of NaN, which a maximum passes over
  a.y = isinf(m) ? a.y + b.y : a.y * ex2((a.x - m) * kLog2e) + b.y * ex2((b.x - m) * kLog2e);
  a.x = m;
}

template <typename T, int V>
__global__ void __launch_bounds__(32 * kJoinRows)
    join_kernel(const float2* __restrict__ parts, uint64_t ld, uint32_t nparts, const Taken Q, const T* __restrict__ w,
                uint64_t ldw, uint32_t d, float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ float2 part[kJoinRows][kJoinRows];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = threadIdx.x % kJoinRows, p0 = threadIdx.x / kJoinRows;
  grid_wait();
  grid_go();
  const uint32_t count = (uint32_t)__ldg(Q.count + 1), row0 = blockIdx.x * kJoinRows, c = row0 + warp;
  if (row0 >= count) return;
  float dot = 0.0f;
  const int32_t target = c < count ? __ldg(Q.target + c) : -1;
  if (target >= 0) dot = target_dot<T, V>(reinterpret_cast<const T*>(Q.h) + (uint64_t)c * Q.ld, w + (uint64_t)target * ldw, d);
  float2 a = make_float2(-INFINITY, 0.0f);
  const bool in = row0 + r < count;
  for (uint32_t p = p0; p < nparts; p += 32 * kJoinAhead) {
    float2 b[kJoinAhead];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u)
      b[u] = in && p + u * 32 < nparts ? __ldcs(parts + (p + u * 32) * ld + row0 + r) : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) join(a, b[u]);
  }
#pragma unroll
  for (int o = kJoinRows; o < 32; o *= 2)
    join(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o)));
  if (lane < kJoinRows) part[warp][lane] = a;
  dot = warp_sum(dot);
  __syncthreads();
  if (c < count && lane == 0) {
    float2 s = part[0][warp];
#pragma unroll
    for (int q = 1; q < kJoinRows; ++q) join(s, part[q][warp]);
    const int32_t row = __ldg(Q.list + c);
    if (target < 0) {  // s is of all the vocabulary
      loss[row] = 0.0f;
      if (lse) lse[row] = s.x + logf(s.y);
      return;
    }
    const float u = fmaxf(s.x, dot);
    if (isinf(u)) {  // as the limits are: lse is infinite, and so is the loss unless the target's logit is too
      const float sum = isnan(s.y) || isnan(dot) ? NAN : u;
      loss[row] = sum - dot;
      if (lse) lse[row] = sum;
      return;
    }
    const float others = s.y == 0.0f ? 0.0f : s.y * ex2((s.x - u) * kLog2e);
    const float more = log1pf(others + (ex2((dot - u) * kLog2e) - 1.0f));
    loss[row] = (u - dot) + more;
    if (lse) lse[row] = u + more;
  }
}

// ---- backward ------------------------------------------------------------------------

// f16 has no room for a mean's small gradients: dl is held times 2^e, the power
// of two that brings the largest |g| to 2^14, so that p down to 2^-39 still counts
// for it, and the products divide by it again. bf16 has f32's range.
__device__ __forceinline__ uint32_t scale_exponent(const unsigned* most) {
  const uint32_t e = __ldg(most) >> 23;  // |g| = 2^(e - 127) times 1 to 2
  return e == 255 ? 127u : min(253u, 127 + 14 + 127 - e);
}
__device__ __forceinline__ float scale_up(const unsigned* most) {
  return most ? __uint_as_float(scale_exponent(most) << 23) : 1.0f;
}
__device__ __forceinline__ float scale_down(const unsigned* most) {
  return most ? __uint_as_float((254u - scale_exponent(most)) << 23) : 1.0f;
}

// A tile of logits to dl, 16-bit, rows at stride ld (a multiple of 8). This is the one
// rounding to 16 bits between the logits and the gradients: half a step of dl,
// which the tensor cores take no wider.
template <typename T>
struct GradientTile {
  static constexpr int kRun = kLogitRun;
  T* dl;
  uint64_t ld;
  const int32_t* target;
  const float* lse;
  const float* g;
  const float* missing;
  const unsigned* most;
  uint32_t v0;

  __device__ __forceinline__ void put(const ProductArgs& P, const Job& j, float (&l)[kHalfTokens], uint32_t lane0,
                                      uint32_t from) const {
    const uint32_t lane = lane0 + (threadIdx.x & 31);
    const bool in = lane < (uint32_t)__ldg(P.lane_count);
    const uint32_t to = min(from + kHalfTokens, j.cols);
    const int32_t mine = in ? __ldg(target + lane) - (int32_t)(v0 + j.col0) : -1;
    const float base = in ? -__ldg(lse + lane) * kLog2e : 0.0f, c = in ? __ldg(g + lane) * scale_up(most) : 0.0f,
                less = in ? __ldg(missing + lane) : 0.0f;
    T* row = dl + (uint64_t)(in ? lane : 0) * ld + j.col0;
#pragma unroll
    for (int q = 0; q < kHalfTokens / 32; ++q) {
      const uint32_t j0 = from + q * 32;
      if (j0 >= to) break;
      float f[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = ex2(__fmaf_rn(l[q * 32 + i], kLog2e, base));
      const uint32_t hit = (uint32_t)(mine - (int32_t)j0);
      if (any_of(hit < 32)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = hit == i ? less : f[i];
      }
      if (in) {
        // sixteen at a time, whole sectors (dl, its rows and j0 lie on 32 bytes): what lies behind the piece's last
        // column is dl's own row
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
          if (j0 + i >= to) break;
          float v[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = f[i + k] * c;
          Pack<T, 16> o;
          o.set(v);
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + j0 + i), "r"(o.w[0]), "r"(o.w[1]),
                       "r"(o.w[2]), "r"(o.w[3]), "r"(o.w[4]), "r"(o.w[5]), "r"(o.w[6]), "r"(o.w[7])
                       : "memory");
        }
      }
    }
  }
};

// A gradient's tile. ADD: the f32 sums of the pieces before, at the same places of
// `sums`, are added first. place: where column j's row goes (null: j itself).
template <typename T, bool ADD>
struct SumsTile {
  static constexpr int kRun = 0;
  T* out;
  const float* sums;
  const int32_t* place;
  const unsigned* most;  // where not null, the values are divided by dl's scale
  uint64_t ld, lds, ldp;  // rows of out and of sums, parts
  bool wide;              // see StoreTile

  __device__ __forceinline__ void put(const ProductArgs& P, const Job& j, uint32_t taddr, uint32_t lane0, uint32_t from,
                                      uint32_t to, uint8_t* scratch) const {
    const uint32_t lane = lane0 + (threadIdx.x & 31);
    const bool in = lane < P.lanes, zero = j.depth == 0;
    const uint32_t l = in ? lane : 0;
    to = min(to, j.cols);
    const float down = scale_down(most);
    if constexpr (sizeof(T) == 2 && !ADD) {
      if (wide) {
        auto row = [&](uint32_t col) {
          const uint64_t r = j.col0 + col;
          return out + (place ? (uint64_t)__ldg(place + r) : r) * ld + lane0;
        };
        const int left = (int)(P.lanes - lane0);
        if (most)
          put_turned<T, true>(taddr, from, to, left, zero, down, scratch, row);
        else
          put_turned<T, false>(taddr, from, to, left, zero, 1.0f, scratch, row);
        return;
      }
    }
    for (uint32_t j0 = from; j0 < to; j0 += 16) {
      const uint32_t n = min(16u, to - j0);
      float g[16];
      if (ADD) {
        const float* s = sums + (uint64_t)j.part * ldp + (uint64_t)(j.col0 + j0) * lds + l;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = in && i < n ? s[i * lds] : 0.0f;
      }
      float f[16];
      tmem_ld16f(taddr + j0, f);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = ((zero ? 0.0f : f[i]) + (ADD ? g[i] : 0.0f)) * down;
      if (place) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (in && i < n) out[(uint64_t)__ldg(place + j.col0 + j0 + i) * ld + l] = from_f32<T>(f[i]);
      } else {
        T* c = out + (uint64_t)j.part * ldp + (uint64_t)(j.col0 + j0) * ld + l;
        if (n == 16) {
          if (in) put16(c, ld, f);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (in && i < n) c[i * ld] = from_f32<T>(f[i]);
        }
      }
    }
  }
};

// dh where its sums were taken in parts: added in order, rounded once, to its rows.
template <typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const float* __restrict__ sums, uint32_t parts, uint64_t ldp,
                                                         uint32_t d, const Taken Q, T* __restrict__ dh, uint64_t lddh) {
  grid_wait();
  grid_go();
  const uint32_t count = (uint32_t)__ldg(Q.count + 1);
  const float down = scale_down(Q.most);
  const uint64_t n = (uint64_t)count * d;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
    float s = 0.0f;
#pragma unroll 8
    for (uint32_t p = 0; p < parts; ++p) s += __ldcs(sums + p * ldp + i);
    dh[(uint64_t)__ldg(Q.list + i / d) * lddh + i % d] = from_f32<T>(s * down);
  }
}

// ---- host ------------------------------------------------------------------------------

constexpr uint64_t kPieceBytes = 256ull << 20;  // of dl, and of copied weights, about
constexpr uint64_t kWorkAligned = 16, kStoreAligned = 32;  // what `work` is, and what dl's widest stores need

uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// How a call is cut, and where its scratch lies: offsets from the first 32-byte boundary in `work`.
struct Plan {
  uint64_t ld;              // of h's rows side by side, and of copied weights
  uint32_t piece, pieces;   // of the vocabulary, a multiple of 256
  uint32_t parts;           // of a piece, in dh
  bool copies;              // weights that TMA cannot read
  uint64_t list, count, target, lse, g, missing, most, h, w, sums, dl, bytes;  // offsets
};

bool weights_in_place(const MapalLossSite& s, const void* w) {
  return aligned16(w) && (s.vocab == 1 || s.ldw % 8 == 0);
}

// Whether the targets' logits are taken eight elements at a time.
bool dots_wide(const MapalLossSite& s, const void* w) { return weights_in_place(s, w) && s.d % 8 == 0; }

Plan plan_of(const MapalLossSite& s, bool grad, bool copies, int sms) {
  Plan p{};
  p.ld = up(s.d, 8);
  p.copies = copies;
  // The vocabulary in pieces of equal size: forward only where weights are copied.
  uint64_t most = up(s.vocab, 256);
  if (copies) most = std::min(most, std::max<uint64_t>(256, kPieceBytes / 2 / p.ld / 256 * 256));
  if (grad) most = std::min(most, std::max<uint64_t>(256, kPieceBytes / 2 / std::max<uint64_t>(s.rows, 1) / 256 * 256));
  p.pieces = (uint32_t)((s.vocab + most - 1) / most);
  p.piece = (uint32_t)up((s.vocab + p.pieces - 1) / p.pieces, 256);
  p.pieces = (uint32_t)((s.vocab + p.piece - 1) / p.piece);
  // dh has rows x d outputs, which may be few tiles: the sum over a piece is cut into the
  // parts that take the least, counted in the time of a block of 64 (270 ns, 2 MB from
  // HBM): a tile's blocks and 8 for its ends, in waves; a part's sums, written and read;
  // and half a block for each that the join adds in turn.
  p.parts = 1;
  if (grad) {
    const uint64_t tiles = up(s.rows, 256) / 256 * (up(s.d, 256) / 256), at_once = sms / 2, blocks = p.piece / kStepK;
    uint64_t least = ~0ull;
    for (uint32_t n = 1; n <= 64 && blocks / n >= 8; ++n) {
      const uint64_t sums = n > 1 ? n * (s.rows * s.d * 8 >> 21) + n / 2 : 0;
      const uint64_t cost = (tiles * n + at_once - 1) / at_once * ((blocks + n - 1) / n + 8) + sums;
      if (cost < least) {
        least = cost;
        p.parts = n;
      }
    }
  }
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  p.list = take(4 * s.rows);
  p.count = take(8);
  p.target = take(4 * s.rows);
  p.h = take(2 * s.rows * p.ld);
  if (copies) p.w = take(2ull * p.piece * p.ld);
  if (grad) {
    p.lse = take(4 * s.rows);
    p.g = take(4 * s.rows);
    p.missing = take(4 * s.rows);
    p.most = take(4);
    p.dl = take(2 * s.rows * p.piece);
    if (p.pieces > 1 || p.parts > 1) p.sums = take(4 * s.rows * s.d * p.parts);
  } else {
    p.sums = take(8 * s.rows * (up(s.vocab, 256) / 128));
  }
  p.bytes = at + (kStoreAligned - kWorkAligned);
  return p;
}

int check_site(const MapalLossSite* s) {
  if (!s) return set_error(MAPAL_ERR_INVALID, "site is null");
  if (s->dtype != MAPAL_DTYPE_F16 && s->dtype != MAPAL_DTYPE_BF16)
    return set_error(MAPAL_ERR_INVALID, "rows and weights are f16 or bf16");
  if (s->vocab == 0 || s->d == 0) return set_error(MAPAL_ERR_INVALID, "no vocabulary, or rows of no elements");
  const uint64_t most = 0x7fffff00ull;
  if (s->rows > most || s->vocab > most || s->d > most)
    return set_error(MAPAL_ERR_UNSUPPORTED, "rows, vocab or d over 2^31 - 256");
  if (!rows_ok(s->rows, s->d, s->ldh, 2) || !rows_ok(s->vocab, s->d, s->ldw, 2) || !rows_ok(s->rows, s->d, s->lddh, 2) ||
      !rows_ok(s->vocab, s->d, s->lddw, 2))
    return set_error(MAPAL_ERR_INVALID, "a row stride is shorter than a row, or too long");
  // scratch of rows x vocab and of rows x d is counted in 64 bits; TMA takes strides below 2^38
  if (s->ldw >= 1ull << 37 || s->vocab * s->ldw >= 1ull << 38 || s->rows * up(s->d, 8) >= 1ull << 38)
    return set_error(MAPAL_ERR_UNSUPPORTED, "an operand over 2^38 elements");
  return 0;
}

struct Call {
  DeviceSlot& D;
  const MapalLossSite& s;
  const Plan p;
  uint8_t* work;
  Taken q;

  template <typename T = uint8_t>
  T* at(uint64_t offset) const {
    return reinterpret_cast<T*>(work + offset);
  }
  Call(DeviceSlot& d, const MapalLossSite& site, const Plan& plan, void* w, bool grad)
      : D(d), s(site), p(plan), work(reinterpret_cast<uint8_t*>(up((uintptr_t)w, kStoreAligned))) {
    q = {at<int32_t>(p.list), at<int32_t>(p.count), at<int32_t>(p.target), at<float>(p.lse), at<float>(p.g), at<float>(p.missing),
         grad && s.dtype == MAPAL_DTYPE_F16 ? at<unsigned>(p.most) : nullptr, at<uint16_t>(p.h), p.ld};
  }

  template <typename T>
  int take(TakeArgs a, const void* h, const void* w, const int32_t* targets) const {
    a.h = static_cast<const uint16_t*>(h);
    a.w = w;
    a.targets = targets;
    a.ldh = s.ldh;
    a.ldw = s.ldw;
    a.wide = dots_wide(s, w);
    a.lddh = s.lddh;
    a.rows = s.rows;
    a.d = s.d;
    a.vocab = (uint32_t)s.vocab;
    a.aligned = aligned16(h) && (s.rows == 1 || s.ldh % 8 == 0);
    a.trap = D.trap;
    const uint64_t blocks = std::min<uint64_t>((s.rows + 3) / 4, 8ull * D.prof.sm_count);
    a.chunk = (uint32_t)((s.rows + blocks - 1) / blocks);
    return launch_rows(take_rows_kernel<T>, (unsigned)((s.rows + a.chunk - 1) / a.chunk), kTakeThreads, 0, D.stream, 1, a, q);
  }
  // The weights of a piece where TMA can read them.
  int weights(const void* w, uint32_t v0, uint32_t n, const void** out, uint64_t* ld) const {
    const uint16_t* from = static_cast<const uint16_t*>(w) + v0 * s.ldw;
    *out = from;
    *ld = s.ldw;
    if (!p.copies) return 0;
    *out = at(p.w);
    *ld = p.ld;
    const uint64_t words = (uint64_t)n * (p.ld / 8);
    return launch_rows(copy_weights_kernel, stream_grid(words, 256, D.prof.sm_count, 8), 256, 0, D.stream, 1, from, s.ldw, n,
                       (uint32_t)s.d, at<uint16_t>(p.w), (uint32_t)p.ld);
  }
  ProductArgs args() const {
    ProductArgs P{};
    P.trap = D.trap;
    P.groups = 1;
    P.parts = 1;
    P.bf16 = s.dtype == MAPAL_DTYPE_BF16;
    return P;
  }
  // Logits of all rows and n of the vocabulary, through `out`.
  template <typename Out>
  int logits(const void* w, uint64_t ldw, uint32_t n, const Out& out) const {
    ProductArgs P = args();
    P.m = n;
    P.lanes = (uint32_t)s.rows;
    P.lane_count = q.count + 1;
    P.depth = (uint32_t)s.d;
    return launch_product_pair<kForward, false, false>(D, {q.h, w, p.ld, 0, ldw, s.rows, s.d, s.d}, P, out);
  }
};

template <typename T>
int forward(const Call& c, const void* h, const void* w, const int32_t* targets, float* loss, float* lse) {
  const MapalLossSite& s = c.s;
  TakeArgs a{};
  a.loss_out = loss;
  a.all = lse != nullptr;
  MAPAL_TRY(c.take<T>(a, h, w, targets));
  float2* parts = c.template at<float2>(c.p.sums);
  for (uint32_t i = 0; i < c.p.pieces; ++i) {
    const uint32_t v0 = i * c.p.piece, n = (uint32_t)std::min<uint64_t>(c.p.piece, s.vocab - v0);
    const void* from;
    uint64_t ldw;
    MAPAL_TRY(c.weights(w, v0, n, &from, &ldw));
    MAPAL_TRY(c.logits(from, ldw, n, SumTile{parts, s.rows, c.q.target, v0, v0 / 128}));
  }
  const uint32_t nparts = (uint32_t)(up(s.vocab, 256) / 128);
  const unsigned blocks = (unsigned)((s.rows + kJoinRows - 1) / kJoinRows);
  auto go = [&](auto kernel) {
    return launch_rows(kernel, blocks, 32 * kJoinRows, 0, c.D.stream, 1, parts, s.rows, nparts, c.q,
                       static_cast<const T*>(w), s.ldw, (uint32_t)s.d, loss, lse);
  };
  return dots_wide(s, w) ? go(join_kernel<T, 8>) : go(join_kernel<T, 1>);
}

template <typename T>
int backward(const Call& c, const void* h, const void* w, const int32_t* targets, const float* lse, const float* dloss,
             void* dh, void* dw) {
  const MapalLossSite& s = c.s;
  const Plan& p = c.p;
  if (c.q.most) MAPAL_CUDA(cudaMemsetAsync(c.q.most, 0, 4, c.D.stream));
  TakeArgs a{};
  a.lse = lse;
  a.dloss = dloss;
  a.dh = static_cast<uint16_t*>(dh);
  a.grad = 1;
  MAPAL_TRY(c.take<T>(a, h, w, targets));
  T* dl = c.template at<T>(p.dl);
  float* sums = c.template at<float>(p.sums);
  const uint64_t ldp = s.rows * s.d;
  for (uint32_t i = 0; i < p.pieces; ++i) {
    const uint32_t v0 = i * p.piece, n = (uint32_t)std::min<uint64_t>(p.piece, s.vocab - v0);
    const void* from;
    uint64_t ldw;
    MAPAL_TRY(c.weights(w, v0, n, &from, &ldw));
    MAPAL_TRY(c.logits(from, ldw, n, GradientTile<T>{dl, p.piece, c.q.target, c.q.lse, c.q.g, c.q.missing, c.q.most, v0}));
    ProductArgs P = c.args();
    P.offsets = c.q.count;
    P.m = (uint32_t)s.rows;
    P.lanes = (uint32_t)s.d;
    if (dw) {
      P.cols = n;
      const SumsTile<T, false> out{static_cast<T*>(dw) + v0 * s.lddw, nullptr, nullptr, c.q.most, s.lddw, 0, 0, aligned16(dw) && s.lddw % 8 == 0};
      MAPAL_TRY((launch_product_pair<kGradW, false, false>(c.D, {c.q.h, dl, p.ld, 0, p.piece, s.rows, s.d, n}, P, out)));
    }
    if (dh) {
      P.depth = n;
      P.parts = p.parts;
      const Operands o{from, dl, ldw, 0, p.piece, n, s.d, n};
      T* to = static_cast<T*>(dh);
      const bool wide = aligned16(dh) && s.lddh % 8 == 0;
      if (p.parts == 1 && i + 1 == p.pieces) {
        if (p.pieces == 1)
          MAPAL_TRY((launch_product_pair<kGradX, false, false>(c.D, o, P, SumsTile<T, false>{to, nullptr, c.q.list, c.q.most, s.lddh, 0, 0, wide})));
        else
          MAPAL_TRY((launch_product_pair<kGradX, false, false>(c.D, o, P, SumsTile<T, true>{to, sums, c.q.list, c.q.most, s.lddh, s.d, 0, false})));
      } else if (i == 0) {
        MAPAL_TRY((launch_product_pair<kGradX, false, false>(c.D, o, P, SumsTile<float, false>{sums, nullptr, nullptr, nullptr, s.d, 0, ldp, false})));
      } else {
        MAPAL_TRY((launch_product_pair<kGradX, false, false>(c.D, o, P, SumsTile<float, true>{sums, sums, nullptr, nullptr, s.d, s.d, ldp, false})));
      }
    }
  }
  if (dh && p.parts > 1)
    MAPAL_TRY(launch_rows(join_parts_kernel<T>, stream_grid(ldp, 256, c.D.prof.sm_count, 8), 256, 0, c.D.stream, 1, sums,
                          p.parts, ldp, (uint32_t)s.d, c.q, static_cast<T*>(dh), s.lddh));
  return 0;
}

int check_work(const Plan& p, const void* work, uint64_t bytes) {
  if (bytes < p.bytes || !work)
    return set_error(MAPAL_ERR_INVALID, "work is shorter than mapal_gpu_linear_loss_workspace says for these arrays");
  if ((uintptr_t)work & (kWorkAligned - 1)) return set_error(MAPAL_ERR_INVALID, "work is not on a 16-byte boundary");
  return 0;
}

}  // namespace

extern "C" int mapal_gpu_linear_loss_workspace(MapalGpuCtx* ctx, const MapalLossSite* site, const void* w, int grad,
                                               uint64_t* bytes) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site));
    if (!bytes) return set_error(MAPAL_ERR_INVALID, "bytes is null");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    const bool copies = !weights_in_place(*site, w);
    const int sms = ctx->dev[0].prof.sm_count;
    *bytes = plan_of(*site, false, copies, sms).bytes;
    if (grad) *bytes = std::max(*bytes, plan_of(*site, true, copies, sms).bytes);
    return 0;
  });
}

extern "C" int mapal_gpu_linear_loss(MapalGpuCtx* ctx, const MapalLossSite* site, const void* h, const void* w,
                                     const int32_t* targets, float* loss, float* lse, void* work, uint64_t work_bytes) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site));
    const MapalLossSite& s = *site;
    if (s.rows == 0) return 0;
    if (!h || !w || !targets || !loss) return set_error(MAPAL_ERR_INVALID, "null h, w, targets or loss");
    if (((uintptr_t)h | (uintptr_t)w) & 1 || ((uintptr_t)targets | (uintptr_t)loss | (uintptr_t)lse) & 3)
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    const Plan p = plan_of(s, false, !weights_in_place(s, w), D.prof.sm_count);
    MAPAL_TRY(check_work(p, work, work_bytes));
    const Call c(D, s, p, work, false);
    if (s.dtype == MAPAL_DTYPE_F16)
      MAPAL_TRY(forward<__half>(c, h, w, targets, loss, lse));
    else
      MAPAL_TRY(forward<__nv_bfloat16>(c, h, w, targets, loss, lse));
    return finish(ctx, 0, true);
  });
}

extern "C" int mapal_gpu_linear_loss_grad(MapalGpuCtx* ctx, const MapalLossSite* site, const void* h, const void* w,
                                          const int32_t* targets, const float* lse, const float* dloss, void* dh, void* dw,
                                          void* work, uint64_t work_bytes) {
  return guarded([&]() -> int {
    MAPAL_TRY(check_site(site));
    const MapalLossSite& s = *site;
    if (!dh && !dw) return 0;
    if (s.rows && (!h || !w || !targets || !lse)) return set_error(MAPAL_ERR_INVALID, "null h, w, targets or lse");
    // a piece's dw is written before its w has gone into dh; h is gathered before anything is written
    if (s.rows && ((dw && (dw == h || dw == dh || (dh && dw == w))) || (dh && (dh == w || (dh == h && s.rows > 1 && s.lddh != s.ldh)))))
      return set_error(MAPAL_ERR_INVALID, "dh or dw is an array that the call reads");
    if (((uintptr_t)h | (uintptr_t)w | (uintptr_t)dh | (uintptr_t)dw) & 1 ||
        ((uintptr_t)targets | (uintptr_t)lse | (uintptr_t)dloss) & 3)
      return set_error(MAPAL_ERR_INVALID, "a pointer is not aligned to its type");
    const OnDevice on(ctx);
    MAPAL_TRY(on.rc);
    DeviceSlot& D = ctx->dev[0];
    if (s.rows == 0) {
      if (dw) MAPAL_TRY(copy_rows(dw, 2 * s.lddw, nullptr, 0, 2 * s.d, s.vocab, D.stream));
      return finish(ctx, 0, false);
    }
    const Plan p = plan_of(s, true, !weights_in_place(s, w), D.prof.sm_count);
    MAPAL_TRY(check_work(p, work, work_bytes));
    const Call c(D, s, p, work, true);
    if (s.dtype == MAPAL_DTYPE_F16)
      MAPAL_TRY(backward<__half>(c, h, w, targets, lse, dloss, dh, dw));
    else
      MAPAL_TRY(backward<__nv_bfloat16>(c, h, w, targets, lse, dloss, dh, dw));
    return finish(ctx, 0, true);
  });
}

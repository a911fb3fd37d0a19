// Log probabilities of chosen elements over ragged segments of logits, with
// the segment's entropy and its largest alternatives, and their gradient.
//
//   lse = log sum_i exp(x_i),  logp = x_t - lse,
//   H   = -sum_i p_i log p_i = log l - s / l,  l = sum e^(x_i - m),
//         s = sum e^(x_i - m) (x_i - m),  m = max x
//   top: the `top` largest x_i (ties to the lowest index) and their x_i - lse
//   dx_i = g_logp [i = t] - p_i (g_logp + sum_k g_top_k)
//          - g_H p_i (log p_i + H) + sum_k g_top_k [i = top_k]
//
// A first pass over a segment keeps (m, l, s) per thread, rescaled when a batch
// raises m. The `top`-th largest of the maxima of up to 64 groups of threads bounds the answer from
// below (that many elements reach it), so a second pass over the segment, which
// the first one left in L2, collects the few elements that reach the bound (24
// on average for the 20 best of a long random row), and each counts those ahead of
// it. Where more reach it than the buffer holds (constant or adversarial rows),
// every warp keeps a sorted list instead, lane r the r-th best. All sums are
// fp32. A segment is read by one CTA, or by the CTAs of a cluster that join
// their statistics and lists through distributed shared memory.
// Bound: HBM on long rows (2,048 x 50,001 bf16: forward 49 us, 4.2 TB/s, its
// exponentials and sums filling 73% of the issue slots; gradient 79 us, 5.2 TB/s
// read and written), latency on short ones (4,096 x 850 fp32 with the 8 best: 14
// and 10 us; 16 x 131,071 bf16 with the 20 best: 15 us, of which one pass over
// 128 CTAs, the bound, the second pass and two cluster barriers). Elements of
// -inf (masked moves) have p = 0 and are never listed; a segment without any
// finite element has lse = logp = -inf, H = 0.
#include <cooperative_groups.h>

#include "common.cuh"
#include "sm100.cuh"

namespace mb {
namespace logp {

using sm100::add2;
using sm100::fma2;
using sm100::mul2;

constexpr int kMaxThreads = 256;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxTop = 32;     // one list entry per lane
constexpr int kMaxSplit = 8;    // CTAs per segment (a portable cluster)
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_(float x) { return ex2(x * kLog2e); }  // e^x for x <= 0

// Softmax statistics relative to the running maximum.
struct Stat {
  float m, l, s;
  __device__ __forceinline__ void raise(float to) {  // to > m
    if (l > 0.f) {
      const float d = m - to, f = exp_(d);
      s = f > 0.f ? (s + d * l) * f : 0.f;
      l *= f;
    }
    m = to;
  }
  __device__ __forceinline__ void merge(Stat o) {
    if (o.m > m) raise(o.m);
    else if (m > o.m) o.raise(m);
    l += o.l;
    s += o.s;
  }
};

// A candidate as one sortable word: the value's order (the two zeros alike),
// then the lower rank. 0 stands for none (no finite value maps to it). Ranks
// have 32 bits; longer segments are refused.
__device__ __forceinline__ unsigned long long key_of(float v, int64_t rank) {
  const uint32_t u = __float_as_uint(v + 0.f);
  const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)order << 32 | (uint32_t)~(uint32_t)rank;
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int64_t rank_of(unsigned long long key) { return (int64_t)(uint32_t)~(uint32_t)key; }

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};

// The elements of 16-byte vector `vec` (counted from `base`, the aligned
// address at or below the array) as floats; those outside [lo, hi) read -inf.
template <typename T>
__device__ __forceinline__ void load_masked(const T* base, int64_t vec, int64_t lo, int64_t hi, float* out) {
  constexpr int N = Vec<T>::N;
  const int64_t e = vec * N;
  if (e >= lo && e + N <= hi) {
    load_vec<N>(base + e, out);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = e + i >= lo && e + i < hi ? to_f(base[e + i]) : -INFINITY;
  }
}

constexpr int kCandidates = kMaxWarps * kMaxTop;  // one per warp and list entry, one per cluster CTA and list entry
constexpr int kGroups = 64;                       // threads' maxima are joined to at most as many
constexpr int U = 2;                              // vectors in flight per thread beside the one in use

// One part of a segment as 16-byte vectors from the aligned address at or below
// the array's start: whole vectors [vb, ve), and the segment's first and last
// vector where it does not fill them (read by the first and last part).
struct Span {
  int64_t lo, hi;      // the segment's elements, from the aligned base
  int64_t vb, ve;
  int64_t head, tail;  // vector or -1
};
template <typename T>
__device__ __forceinline__ Span span_of(int64_t a, int64_t b, int64_t shift, int part, int split) {
  constexpr int N = Vec<T>::N;
  Span s{a + shift, b + shift, 0, 0, -1, -1};
  if (b <= a) return s;
  int64_t first = s.lo / N, last = (s.hi - 1) / N;
  const bool head = s.lo > first * N || s.hi < (first + 1) * N, tail = last > first && s.hi < (last + 1) * N;
  if (head && part == 0) s.head = first;
  if (tail && part == split - 1) s.tail = last;
  first += head;
  last -= tail;
  const int64_t n = max(last + 1 - first, (int64_t)0);
  s.vb = first + n * part / split;
  s.ve = first + n * (part + 1) / split;
  return s;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& raw, float* x) {
  if constexpr (sizeof(T) == 4) {
    x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y), x[2] = __uint_as_float(raw.z),
    x[3] = __uint_as_float(raw.w);
  } else {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// body(x, v) for every vector of the part; the elements of a partly filled one
// outside the segment are -inf. A thread keeps U loads in flight beside the
// vector that it works on (2,048 x 50,001 bf16, forward and gradient: 58 and 94 us
// with none, 89 and 127 us with four loads before their use, 51 and 85 us so;
// eight CTAs per SM then take the gradient to 79 us, six the forward to 49 us).
template <typename T, typename Body>
__device__ __forceinline__ void scan(const T* base, const Span& s, Body body) {
  constexpr int N = Vec<T>::N;
  const uint4* vecs = reinterpret_cast<const uint4*>(base);
  const int step = blockDim.x;
  int64_t v = s.vb + threadIdx.x;
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v + u * step < s.ve) raw[u] = __ldg(vecs + v + u * step);
  if (threadIdx.x < 2) {  // the edges, while the first loads are on their way
    const int64_t e = threadIdx.x == 0 ? s.head : s.tail;
    if (e >= 0) {
      float x[N];
      load_masked(base, e, s.lo, s.hi, x);
      body(x, e);
    }
  }
  while (v < s.ve) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v >= s.ve) break;
      float x[N];
      unpack<T>(raw[u], x);
      if (v + U * step < s.ve) raw[u] = __ldg(vecs + v + U * step);
      body(x, v);
      v += step;
    }
  }
}

// A CTA's list buffers.
struct Lists {
  unsigned long long cand[kCandidates];
  unsigned long long out[kMaxTop];
  float maxima[kGroups];
  int bound;  // an ordered float
  int count;
};

// Floats in the order of ints.
__device__ __forceinline__ int ordered(float v) {
  const int i = __float_as_int(v);
  return i < 0 ? i ^ 0x7fffffff : i;
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i < 0 ? i ^ 0x7fffffff : i); }

// out = the `top` best of the n candidates: each counts those ahead of it.
__device__ __forceinline__ void rank_candidates(Lists& ls, int n, int top) {
  if (threadIdx.x < top) ls.out[threadIdx.x] = 0;
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const unsigned long long mine = ls.cand[c];
    int ahead = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) ahead += ls.cand[j] > mine;
    if (mine != 0 && ahead < top) ls.out[ahead] = mine;
  }
  __syncthreads();
}

// The best of vectors [vb, ve) by a sorted list per warp (lane r holds the
// r-th best), for rows that overflow the candidates: every element past the
// list's last entry is inserted.
template <typename T>
__device__ __noinline__ void warp_lists(Lists& ls, const T* base, int64_t vb, int64_t ve, int64_t lo, int64_t hi,
                                        int top) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long best = 0;
  float thr = -INFINITY;
  for (int64_t w0 = vb + warp * 32; w0 < ve; w0 += blockDim.x) {
    float x[N];
    if (w0 + lane < ve) {
      load_masked(base, w0 + lane, lo, hi, x);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = -INFINITY;
    }
    float bm = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) bm = fmaxf(bm, x[i]);
    // ranks ascend over a warp's steps, lanes and elements: an equal value
    // that comes later is behind those listed
    unsigned todo = __ballot_sync(0xffffffffu, bm > thr);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      const int64_t e = (w0 + src) * N - lo;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = __shfl_sync(0xffffffffu, x[i], src);
        if (v > thr) {
          const unsigned long long key = key_of(v, e + i);
          const int pos = __popc(__ballot_sync(0xffffffffu, best > key));
          const unsigned long long up = __shfl_up_sync(0xffffffffu, best, 1);
          if (lane >= pos) best = lane == pos ? key : up;
          const unsigned long long last = __shfl_sync(0xffffffffu, best, top - 1);
          thr = last ? value_of(last) : -INFINITY;
        }
      }
    }
  }
  __syncthreads();
  if (lane < top) ls.cand[warp * top + lane] = best;
  __syncthreads();
}

// Ranks have 32 bits.
__device__ __forceinline__ bool malformed(int64_t a, int64_t b, int64_t n) {
  return a < 0 || b < a || b > n || b - a > 0xffffffffLL;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kMaxThreads, TOP ? 4 : 6) forward_kernel(
    const T* __restrict__ logits, int64_t n, const int64_t* __restrict__ offsets, const int64_t* __restrict__ ranks,
    int top, int split, float* __restrict__ lse, float* __restrict__ logp, float* __restrict__ entropy,
    int64_t* __restrict__ top_ranks, float* __restrict__ top_logp) {
  constexpr int N = Vec<T>::N;
  __shared__ Stat stats[kMaxWarps];
  __shared__ Stat cta_stat;
  __shared__ __align__(16) uint8_t list_space[TOP ? sizeof(Lists) : 16];
  Lists& ls = *reinterpret_cast<Lists*>(list_space);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int64_t p = blockIdx.x / split;
  const int part = blockIdx.x % split;
  int64_t a = offsets[p], b = offsets[p + 1];
  if (malformed(a, b, n)) {
    if (tid == 0) report(ERR_RUN_BOUND);
    a = b = 0;
  }
  const int64_t shift = (int64_t)(reinterpret_cast<uintptr_t>(logits) & 15) / (int64_t)sizeof(T);
  const T* base = logits - shift;
  const Span span = span_of<T>(a, b, shift, part, split);
  Stat st{kLowest, 0.f, 0.f};
  scan(base, span, [&](const float* x, int64_t) {
    float bm = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) bm = fmaxf(bm, x[i]);
    if (bm > st.m) st.raise(bm);
    const float2 down = make_float2(-st.m, -st.m), unit = make_float2(kLog2e, kLog2e);
    float2 l = make_float2(st.l, 0.f), s = make_float2(st.s, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 d = add2(make_float2(x[i], x[i + 1]), down), y = mul2(d, unit);
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      l = add2(l, e);
      s = fma2(e, make_float2(fmaxf(d.x, kLowest), fmaxf(d.y, kLowest)), s);  // e = 0 at d = -inf
    }
    st.l = l.x + l.y;
    st.s = s.x + s.y;
  });
  const int per_group = max(1, (int)blockDim.x / kGroups), groups = blockDim.x / per_group;
  if (TOP) {
    float top_v = st.l > 0.f ? st.m : -INFINITY;
    for (int o = per_group >> 1; o > 0; o >>= 1) top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
    if (tid % per_group == 0) ls.maxima[tid / per_group] = top_v;
    if (tid == 0) {
      ls.bound = ordered(INFINITY);
      ls.count = 0;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.l, o),
               __shfl_xor_sync(0xffffffffu, st.s, o)};
    st.merge(other);
  }
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < warps; ++w) st.merge(stats[w]);
    cta_stat = st;
  }
  if (TOP) {
    // the bound: the smallest maximum that fewer than `top` are above (-inf
    // where fewer groups than that hold an element)
    if (tid < groups) {
      const float mine = ls.maxima[tid];
      int ahead = 0;
#pragma unroll 4
      for (int j = 0; j < groups; j += 4) {
        const float4 o = *reinterpret_cast<const float4*>(ls.maxima + j);
        ahead += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      }
      if (ahead < top) atomicMin(&ls.bound, ordered(mine));
    }
    __syncthreads();
    const float bound = groups < top ? -INFINITY : unordered(ls.bound);
    scan(base, span, [&](const float* x, int64_t v) {
      float bm = x[0];
#pragma unroll
      for (int i = 1; i < N; ++i) bm = fmaxf(bm, x[i]);
      if (bm >= bound && bm > -INFINITY) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (x[i] >= bound && x[i] > -INFINITY) {
            const int c = atomicAdd(&ls.count, 1);  // the order does not matter: candidates are ranked
            if (c < kCandidates) ls.cand[c] = key_of(x[i], v * N + i - span.lo);
          }
      }
    });
    __syncthreads();
    int found = ls.count;
    if (found > kCandidates) {
      warp_lists(ls, base, span.head >= 0 ? span.head : span.vb, span.tail >= 0 ? span.tail + 1 : span.ve, span.lo,
                 span.hi, top);
      found = warps * top;
    }
    rank_candidates(ls, found, top);
  }
  if (split > 1) {
    auto cluster = cooperative_groups::this_cluster();
    cluster.sync();  // every CTA's statistics and list are written
    if (part == 0) {
      if (tid == 0) {
        for (int c = 1; c < split; ++c) st.merge(*cluster.map_shared_rank(&cta_stat, c));
        cta_stat = st;
      }
      if (TOP)
        for (int c = tid; c < split * top; c += blockDim.x)
          ls.cand[c] = *cluster.map_shared_rank(&ls.out[c % top], c / top);
    }
    cluster.sync();  // the other CTAs' shared memory is read
    if (part != 0) return;
    if (TOP) rank_candidates(ls, split * top, top);
  }
  __syncthreads();
  const Stat all = cta_stat;
  const bool none = !(all.l > 0.f) && all.l == all.l;  // nothing finite (a NaN sum stays a NaN)
  const float logl = logf(all.l);
  if (tid == 0) {
    const int64_t t = ranks ? ranks[p] : -1;
    lse[p] = none ? -INFINITY : all.m + logl;
    entropy[p] = none ? 0.f : logl - all.s / all.l;
    float got = 0.f;  // no chosen element
    if (t >= b - a) report(ERR_INDEX);
    else if (t >= 0) got = none ? -INFINITY : (to_f(logits[a + t]) - all.m) - logl;
    logp[p] = got;
  }
  if (TOP && tid < top) {
    const unsigned long long key = ls.out[tid];
    top_ranks[p * top + tid] = key ? rank_of(key) : -1;
    top_logp[p * top + tid] = key ? (value_of(key) - all.m) - logl : -INFINITY;
  }
}

// A malformed segment reads as empty, in both directions. Its offsets may leave
// elements to no segment at all, whose gradient is zero: this one clears, of
// those between the highest offset so far and its own end, the ones that no well-
// formed segment holds. Offsets that pass an element for the first time do so
// in such a step or in a well-formed segment, so all are written; the first and
// last segment clear what lies outside all offsets. Off the ordinary path: every
// step here reads the offsets, and no element is cleared twice.
template <typename T>
__device__ __forceinline__ void zero_malformed(const int64_t* __restrict__ offsets, int64_t n_segments, int64_t p,
                                            int64_t n, T* __restrict__ grad) {
  __shared__ long long reach, next;
  const long long end = min(max(offsets[p + 1], (int64_t)0), n);
  if (threadIdx.x == 0) reach = 0;
  __syncthreads();
  for (int64_t i0 = p; i0 >= 0; i0 -= blockDim.x) {  // the highest offset so far
    const int64_t i = i0 - threadIdx.x;
    const long long o = i >= 0 ? min(max(offsets[i], (int64_t)0), n) : 0;
    atomicMax(&reach, o);
    if (__syncthreads_or(o >= end)) return;
  }
  long long at = reach;
  while (at < end) {
    __syncthreads();
    if (threadIdx.x == 0) reach = at, next = end;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < n_segments; i += blockDim.x) {
      const long long a = offsets[i], b = offsets[i + 1];
      if (malformed(a, b, n) || b <= at) continue;
      if (a <= at) atomicMax(&reach, b);
      else atomicMin(&next, a);
    }
    __syncthreads();
    const long long held = reach, to = next;
    if (held == at)
      for (long long e = at + threadIdx.x; e < to; e += blockDim.x) grad[e] = from_f<T>(0.f);
    at = held > at ? held : to;
  }
}

template <typename T>
__global__ void __launch_bounds__(kMaxThreads, 8) backward_kernel(
    const T* __restrict__ logits, int64_t n, const int64_t* __restrict__ offsets, const int64_t* __restrict__ ranks,
    int top, int split, const float* __restrict__ lse, const float* __restrict__ entropy,
    const int64_t* __restrict__ top_ranks, const float* __restrict__ g_logp, const float* __restrict__ g_entropy,
    const float* __restrict__ g_top, T* __restrict__ grad) {
  constexpr int N = Vec<T>::N;
  __shared__ int64_t hot_i[kMaxTop + 1];
  __shared__ float hot_g[kMaxTop + 1];
  const int tid = threadIdx.x;
  const int64_t p = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const int64_t a = offsets[p], b = offsets[p + 1];
  // elements outside every segment have no gradient
  if (part == 0) {
    if (p == 0)
      for (int64_t e = tid; e < min(a, n); e += blockDim.x) grad[e] = from_f<T>(0.f);
    if ((p + 1) * split == gridDim.x)
      for (int64_t e = max(b, (int64_t)0) + tid; e < n; e += blockDim.x) grad[e] = from_f<T>(0.f);
  }
  if (malformed(a, b, n)) {
    if (tid == 0) report(ERR_RUN_BOUND);
    if (part == 0) zero_malformed(offsets, gridDim.x / split, p, n, grad);
    return;
  }
  if (b == a) return;
  // the elements with a gradient of their own: the chosen one, then the listed ones
  if (tid <= top) {
    int64_t i = tid == 0 ? (ranks ? ranks[p] : -1) : top_ranks[p * top + tid - 1];
    if (i >= b - a) {
      report(ERR_INDEX);
      i = -1;
    }
    hot_i[tid] = i;
    hot_g[tid] = i < 0 ? 0.f : tid == 0 ? (g_logp ? g_logp[p] : 0.f) : g_top[p * top + tid - 1];
  }
  __syncthreads();
  float weight = 0.f;
  for (int j = 0; j <= top; ++j) weight += hot_g[j];
  const float z = lse[p], h = entropy[p], gh = g_entropy ? g_entropy[p] : 0.f;
  // dx = -p (weight + g_H (log p + H)), log p = x - lse; a segment without a
  // finite element has no gradient. p = 0 at log p = -inf, whose product needs
  // a finite factor.
  const bool none = z == -INFINITY;
  const float2 down = make_float2(-z, -z), unit = make_float2(kLog2e, kLog2e), slope = make_float2(-gh, -gh);
  const float at0 = -fmaf(gh, h, weight);
  auto grad2 = [&](float x0, float x1) {
    const float2 lp = add2(make_float2(x0, x1), down), y = mul2(lp, unit);
    const float2 pr = make_float2(ex2(y.x), ex2(y.y));
    const float2 g = mul2(pr, fma2(slope, make_float2(fmaxf(lp.x, -1e30f), fmaxf(lp.y, -1e30f)),
                                   make_float2(at0, at0)));
    return none ? make_float2(0.f, 0.f) : g;
  };

  const int64_t shift = (int64_t)(reinterpret_cast<uintptr_t>(logits) & 15) / (int64_t)sizeof(T);
  const T* base = logits - shift;
  T* gbase = grad - shift;
  const Span span = span_of<T>(a, b, shift, part, split);
  scan(base, span, [&](const float* x, int64_t v) {
    float y[N];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 g = grad2(x[i], x[i + 1]);
      y[i] = g.x;
      y[i + 1] = g.y;
    }
    const int64_t e = v * N;
    if (v != span.head && v != span.tail) {
      store_vec<N>(gbase + e, y);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e + i >= span.lo && e + i < span.hi) gbase[e + i] = from_f<T>(y[i]);
    }
  });
  __syncthreads();
  // this part's elements with a gradient of their own; the first of equal
  // indices writes the sum of them all
  if (tid <= top && hot_i[tid] >= 0 && !none) {
    const int64_t i = hot_i[tid], e = span.lo + i, v = e / N;
    bool mine = (v >= span.vb && v < span.ve) || v == span.head || v == span.tail;
    float g = 0.f;
    for (int j = 0; j <= top; ++j)
      if (hot_i[j] == i) {
        if (j < tid) mine = false;
        g += hot_g[j];
      }
    if (mine) gbase[e] = from_f<T>(grad2(to_f(base[e]), 0.f).x + g);
  }
}

// Threads per CTA: about eight vectors a thread at the mean length (a warp of
// its own for rows up to that, which needs no barrier), two where segments
// leave the GPU empty. CTAs per segment: enough to give every SM two where
// segments are few and long, each keeping at least 4096 elements.
struct Shape {
  int threads, split;
};
inline Shape shape(int64_t n, int64_t segments, int vec) {
  const int64_t mean = n / segments;
  int threads = 32;
  while (threads < kMaxThreads && threads * vec * (segments * threads < 148 * 512 ? 2 : 8) < mean) threads *= 2;
  int split = 1;
  while (split < kMaxSplit && segments * split < 2 * 148 && mean / (2 * split) >= 4096) split *= 2;
  return {threads, split};
}

}  // namespace logp
}  // namespace mb

using namespace mb;

extern "C" int mb_log_probs(const void* logits, int dtype, int64_t n, const int64_t* offsets, int64_t n_segments,
                            const int64_t* ranks, int top, float* lse, float* logp, float* entropy,
                            int64_t* top_ranks, float* top_logp, void* stream) {
  MB_REQUIRE(valid_dtype(dtype), "log_probs: bad dtype");
  MB_REQUIRE(n >= 0 && n_segments >= 0, "log_probs: negative size");
  MB_REQUIRE(top >= 0 && top <= logp::kMaxTop, "log_probs: top must be in [0, %d] (got %d)", logp::kMaxTop, top);
  if (n_segments == 0) return MB_OK;
  MB_REQUIRE((n == 0 || logits) && offsets && lse && logp && entropy && (top == 0 || (top_ranks && top_logp)),
             "log_probs: null pointer");
  MB_REQUIRE(aligned(logits, dtype_size(dtype)), "log_probs: logits must be aligned to their type");
  MB_REQUIRE(n_segments <= INT32_MAX / logp::kMaxSplit, "log_probs: too many segments");
  const logp::Shape sh = logp::shape(n, n_segments, 16 / dtype_size(dtype));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_segments * sh.split));
  cfg.blockDim = dim3((unsigned)sh.threads);
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)sh.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = sh.split > 1 ? 1 : 0;
  MB_DISPATCH_T(dtype, T, [&] {
    auto kern = top ? logp::forward_kernel<T, true> : logp::forward_kernel<T, false>;
    (void)cudaLaunchKernelEx(&cfg, kern, (const T*)logits, n, offsets, ranks, top, sh.split, lse, logp, entropy,
                             top_ranks, top_logp);
  });
  return launch_status("log_probs");
}

extern "C" int mb_log_probs_backward(const void* logits, int dtype, int64_t n, const int64_t* offsets,
                                     int64_t n_segments, const int64_t* ranks, int top, const float* lse,
                                     const float* entropy, const int64_t* top_ranks, const float* g_logp,
                                     const float* g_entropy, const float* g_top, void* grad, void* stream) {
  MB_REQUIRE(valid_dtype(dtype), "log_probs_backward: bad dtype");
  MB_REQUIRE(n >= 0 && n_segments >= 0, "log_probs_backward: negative size");
  MB_REQUIRE(top >= 0 && top <= logp::kMaxTop, "log_probs_backward: top must be in [0, %d] (got %d)", logp::kMaxTop,
             top);
  if (n == 0) return MB_OK;
  MB_REQUIRE(grad, "log_probs_backward: null pointer");
  if (n_segments == 0) {  // every element is outside every segment
    (void)cudaMemsetAsync(grad, 0, (size_t)n * dtype_size(dtype), as_stream(stream));
    return launch_status("log_probs_backward");
  }
  MB_REQUIRE(logits && offsets && lse && entropy && (top == 0 || (top_ranks && g_top)),
             "log_probs_backward: null pointer");
  MB_REQUIRE(aligned(logits, dtype_size(dtype)) && ((uintptr_t)logits & 15) == ((uintptr_t)grad & 15),
             "log_probs_backward: logits and grad must be aligned alike");
  MB_REQUIRE(n_segments <= INT32_MAX / logp::kMaxSplit, "log_probs_backward: too many segments");
  const logp::Shape sh = logp::shape(n, n_segments, 16 / dtype_size(dtype));
  const unsigned grid = (unsigned)(n_segments * sh.split);
  // a CTA holds the top + 1 elements with a gradient of their own
  const int threads = sh.threads <= top ? 64 : sh.threads;
  MB_DISPATCH_T(dtype, T, [&] {
    logp::backward_kernel<T><<<grid, threads, 0, as_stream(stream)>>>(
        (const T*)logits, n, offsets, ranks, top, sh.split, lse, entropy, top_ranks, g_logp, g_entropy, g_top,
        (T*)grad);
  });
  return launch_status("log_probs_backward");
}

// Attention with a learned relative position bias by buckets, the parts that
// its CUDA-core and tensor-core kernels share. Per position p, head h, with
// g = h / (heads / kv_heads):
//
//   s_ij = scale q_i . k_j + bias[b_ij, h],  b_ij = map[clamp(c_j - c_i)]
//   P = softmax_j(s) over the keys j < valid[p] whose map entry is not -1
//   out_i = sum_j P_ij v_j,  lse_i = log sum_j exp(s_ij)
//
// c are two-component integer coordinates, clamped per component to the map's
// radii; a row without a key (or past valid[p]) has out = 0, lse = -inf.
#pragma once

#include <atomic>

#include "common.cuh"

namespace mb {
namespace bucket {

constexpr int kMaxMap = 4096;     // map entries (staged in shared memory)
constexpr int kMaxBuckets = 128;  // bias rows
// A bias this low is a mask: the pair is excluded as with -inf, so that a row
// with nothing else reads zero (its probabilities could not be recomputed: the
// log-sum-exp would have lost the sum).
constexpr float kMaskBias = -1e4f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Strides {
  int64_t pos, head, row;
};

struct Args {
  const void *q, *k, *v;
  Strides sq, sk, sv;
  int64_t n_pos, length;
  int heads, kv_heads, dim;
  float scale;
  const float* bias;     // (n_buckets, heads)
  int n_buckets;
  const int32_t* map;    // (2 rq + 1, 2 rr + 1)
  int rq, rr;
  const int32_t* coords; // (n_pos, length, 2), positions c_pos apart
  int64_t c_pos;
  const int32_t* valid;  // (n_pos) or null
  void* out;
  Strides so;
  float* full;           // contiguous (n_pos, heads, length, dim) or null: out before its rounding
  float* lse;            // (n_pos, heads, length) or null
  // backward
  const void* grad;
  Strides sg;
  const float* lse_in;
  float* delta;          // (n_pos, heads, length): dO . out
  float* dq_part;        // per key tile (n_pos, heads, length, dim) sums, or null
  float* dkv_part;       // per split the (dk, dv) sums, or null
  float* bias_part;      // (heads, n_buckets, CTAs per head)
  void *dq, *dk, *dv;    // contiguous
  float* dbias;          // (n_buckets, heads) or null
};

__device__ __forceinline__ int valid_of(const Args& a, int64_t p) {
  if (!a.valid) return (int)a.length;
  const int nv = a.valid[p];
  if (nv >= 0 && nv <= a.length) return nv;
  if (threadIdx.x == 0) report(ERR_INDEX);
  return nv < 0 ? 0 : (int)a.length;
}

// Saturating difference: coordinates may span the whole int32 range.
__device__ __forceinline__ int sub_sat(int a, int b) {
  int d;
  asm("sub.sat.s32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The map entry of a key's offset from a query.
__device__ __forceinline__ int entry_of(const Args& a, int2 query, int2 key) {
  const int x = min(max(sub_sat(key.x, query.x), -a.rq), a.rq) + a.rq;
  const int y = min(max(sub_sat(key.y, query.y), -a.rr), a.rr) + a.rr;
  return x * (2 * a.rr + 1) + y;
}

// The bucket that a map entry names, or -1 for an excluded pair; an entry past
// the table is an index error and excludes the pair too.
__device__ __forceinline__ int checked_bucket(const Args& a, int b) {
  if (b >= a.n_buckets || b < -1) {
    report(ERR_INDEX);
    return -1;
  }
  return b;
}
__device__ __forceinline__ int bucket_of(const Args& a, int entry) { return checked_bucket(a, __ldg(a.map + entry)); }

// A head's bias, in log2 units; -inf for a mask.
__device__ __forceinline__ float bias_of(const Args& a, int bucket, int h) {
  const float b = __ldg(a.bias + (int64_t)bucket * a.heads + h);
  return b <= kMaskBias ? -INFINITY : b * kLog2e;
}

// Every map entry's bucket (-1: excluded) and bias to put(entry, bucket,
// bias), by THREADS threads: the head's bias column passes through `column`
// (n_buckets floats of shared memory), and a thread's map loads are all in
// flight at once, so one global latency is paid. Ends without a barrier.
template <int THREADS, typename Put>
__device__ __forceinline__ void spread_bias(const Args& a, int h, float* column, Put put) {
  constexpr int U = 8;
  const int n = (2 * a.rq + 1) * (2 * a.rr + 1);
  int b[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = threadIdx.x + u * THREADS;
    b[u] = i < n ? __ldg(a.map + i) : -1;
  }
  for (int i = threadIdx.x; i < a.n_buckets; i += THREADS) column[i] = bias_of(a, i, h);
  __syncthreads();
  for (int i0 = threadIdx.x; i0 < n; i0 += U * THREADS) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * THREADS;
      if (i < n) {
        const int k = checked_bucket(a, i0 == threadIdx.x ? b[u] : __ldg(a.map + i));
        put(i, k, k < 0 ? -INFINITY : column[k]);
      }
    }
  }
}

template <typename K>
int configure(K kern, size_t bytes, const char* what) {
  if (bytes <= 48 * 1024) return MB_OK;  // granted without asking
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
    return fail(MB_LAUNCH_FAILED, "%s: %zu bytes of shared memory refused", what, bytes);
  return MB_OK;
}

// The tensor-core forms (bucket_attention_sm100.cu).
bool tc_serves(const Args& a, int dtype);
int tc_forward(const Args& a, cudaStream_t s);
// How the tensor-core backward pass is shared (see bucket_attention_sm100.cu):
// by whole items, or key tiles, how many of them a launch takes (their dQ parts
// are kept together) and the CTAs that share a key tile's queries.
struct BackwardPlan {
  bool whole;
  int64_t tiles, chunk, split;
  int64_t ctas;                 // bias sums kept per (head, bucket)
  int64_t dq_words, dkv_words;  // fp32 workspace words of the parts
};
BackwardPlan backward_plan(int64_t n_pos, int heads, int kv_heads, int head_dim, int64_t length, int dtype);
int tc_backward(const Args& a, const BackwardPlan& plan, cudaStream_t s);

// fp32 words of dQ parts that a caller allows a backward pass (0: the default).
extern std::atomic<int64_t> part_limit;

}  // namespace bucket
}  // namespace mb
